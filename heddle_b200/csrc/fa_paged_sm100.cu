// hb_fa_paged: checks, the workspace and the launches of the paged attention (fa_paged_sm100.cuh).
#include "fa_paged_tiles_sm100.cuh"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <mutex>

#include "host_common.h"

namespace hb {

static std::mutex g_paged_mutex;

static int paged_check(const char* fn, const hb_fa_paged_args* a, bool* empty) {
  if (a == nullptr) return set_error(HB_ERR_BAD_ARG, "%s: args is NULL", fn);
  const hb_kv_cache& c = a->cache;
  const int rc = kv_cache_check(fn, c, empty);
  if (rc != HB_OK) return rc;
  if (a->dtype != HB_BF16 && a->dtype != HB_FP16) return set_error(HB_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are built)", fn, a->dtype);
  if (a->Hq <= 0 || a->Hq % c.Hkv != 0) return set_error(HB_ERR_BAD_ARG, "%s: Hq = %d must be a multiple of Hkv = %d", fn, a->Hq, c.Hkv);
  if (static_cast<int64_t>(c.T) * a->Hq > 0x7fffffffll || static_cast<int64_t>(c.B) * a->Hq > 0x7fffffffll)
    return set_error(HB_ERR_UNSUPPORTED, "%s: T * Hq and B * Hq may not exceed 2^31", fn);
  if (*empty) return HB_OK;
  if (a->q == nullptr || a->o == nullptr) return set_error(HB_ERR_BAD_ARG, "%s: NULL pointer", fn);
  const uint64_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o) |
                        static_cast<uint64_t>(2 * (a->q_stride_t | a->q_stride_h | a->o_stride_t | a->o_stride_h));
  if ((bits & 15u) != 0 || (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0)
    return set_error(HB_ERR_ALIGN, "%s: rows of q and o must be 16-byte aligned, lse 4-byte aligned", fn);
  return HB_OK;
}

// Query rows of a (sequence, KV head) at most, INT_MAX where the call does not say.
static int64_t paged_most_rows(const hb_fa_paged_args* a) {
  const hb_kv_cache& c = a->cache;
  const int64_t group = a->Hq / c.Hkv;
  if (c.starts == nullptr) return group * (c.T / c.B);
  return a->max_tokens > 0 ? group * std::min(a->max_tokens, c.T) : INT_MAX;
}
// Which kernels a call takes and what they need; worked out from the arguments, which hold nothing that is on the device.
struct PagedRoute {
  bool rows_kernel, tiles_kernel;
  int row_limit;              // the tiles kernel has the sequences of more query rows a KV head, the rows kernel the others
  int tile_rows, blocks;      // rows kernel: rows of a row tile, blocks of the grid
  int64_t items;              // tiles kernel: items, blocks of the grid for each
  int splits;
  uint64_t tiles_bytes, bytes;  // of the workspace: the tiles kernel's part, which comes first, and all
};

// Blocks for an item of the tiles kernel: as many as one round of blocks has place for, up to 16, each with three tiles at least of those that
// the page table has room for.  More rounds of smaller blocks cost more than they even out, since a block's start and end take about as
// long as four tiles.  us with 1 | 2 | 4 | 8 blocks an item: B1 Hq32 Hkv8, 128 rows, 4096 keys (8 items) 71.4 | 42.8 | 28.1 | 22.8; 512 rows (16 items) 77 | 48 |
// 32 | 31; B1 Hq32 Hkv2, 128 rows, 20000 keys (2 items) 328 | 169 | 91 | 55 (16: 39); B4, 256 rows, 2000 to 4096 keys (32 items) 77 | 49 | 36 | 44.
constexpr int kPagedMaxSplits = 16;
static int paged_splits(int64_t items, double key_tiles, int sm_count) {
  const int64_t round = items > 0 ? sm_count / items : 1;
  return (int)std::max<int64_t>(1, std::min({round, (int64_t)(key_tiles / 3), (int64_t)kPagedMaxSplits}));
}

// The limit is where 32 keys cost the SMs as much either way, all sequences taken alike: in the rows kernel 375 cycles for every 16 rows,
// dealt out evenly; in the tiles kernel 850 for up to 256, by rounds of whole blocks, or, where items are dealt out to several blocks,
// divided by 0.6 of their number, which is what their starts and the merge leave of it.  us, rows kernel | tiles kernel, Hq32 Hkv8, 2000
// to 4096 keys: B1 64 rows (a KV head) 19 | 23, 128 rows 26 | 23; B4 48 rows 31 | 31, 64 rows 35 | 31, 128 rows 61 | 32; B16 32 rows 51 | 75, 48 rows 70 | 74,
// 64 rows 89 | 74; B64 32 rows 165 | 235, 48 rows 243 | 243.
static int paged_row_limit(int64_t pairs, int64_t most_rows, double key_tiles, int sm_count) {
  int limit = kPagedMaxRows;
  while (limit < most_rows && limit < 4096) {
    const int tiles = limit / kPagedMaxRows + 1;
    const int64_t blocks = pairs * ((tiles * kPagedMaxRows + kPagedBlockRows - 1) / kPagedBlockRows);
    const int splits = paged_splits(blocks, key_tiles, sm_count);
    const double rows_cost = (double)pairs * tiles / sm_count * 375;
    const double tiles_cost = 850 * (splits > 1 ? 1 / std::max(1.0, 0.6 * splits) : (double)((blocks + sm_count - 1) / sm_count));
    if (rows_cost > tiles_cost) break;
    limit += kPagedMaxRows;
  }
  return limit;
}

static PagedRoute paged_route(const hb_fa_paged_args* a, int sm_count) {
  const hb_kv_cache& c = a->cache;
  const int64_t group = a->Hq / c.Hkv, pairs = (int64_t)c.B * c.Hkv, all_rows = group * c.T, most_rows = paged_most_rows(a);
  const double key_tiles = (double)c.max_pages * c.page_size / kTileN;
  PagedRoute r = {};
  r.row_limit = paged_row_limit(pairs, std::min(most_rows, all_rows), key_tiles, sm_count);
  r.tiles_kernel = std::min(most_rows, all_rows) > r.row_limit;
  r.rows_kernel = c.starts != nullptr || !r.tiles_kernel;
  if (r.tiles_kernel) {
    // exactly, or where the device knows only, as many as so many rows can be
    if (c.starts == nullptr) r.items = pairs * ((all_rows / c.B + kPagedBlockRows - 1) / kPagedBlockRows);
    else r.items = c.Hkv * (all_rows / kPagedBlockRows + std::min<int64_t>(c.B, all_rows / (r.row_limit + 1)));
    r.splits = paged_splits(r.items, key_tiles, sm_count);
    if (r.splits > 1) r.tiles_bytes = r.items * (sizeof(PagedParts) + (uint64_t)r.splits * kPagedBlockRows * (c.D + 1) * sizeof(float));
  }
  r.bytes = r.tiles_bytes;
  if (r.rows_kernel) {
    r.tile_rows = most_rows <= 8 ? 8 : kPagedMaxRows;
    // as many blocks as the device holds, and no more than the list can fill: of tiles that the page table has room for
    const bool few = r.tile_rows == 8;
    const int most = sm_count * (c.D == 128 ? (few ? paged_blocks_per_sm<128, 8> : paged_blocks_per_sm<128, 16>)
                                            : (few ? paged_blocks_per_sm<64, 8> : paged_blocks_per_sm<64, 16>));
    const double row_tiles = (double)all_rows / r.tile_rows + c.B;
    const double runs = row_tiles * c.Hkv * paged_places(paged_tiles(c.max_pages * c.page_size, paged_tile(c.D))) / kPagedWarps + 1;
    r.blocks = runs < most ? (int)runs : most;
    r.bytes += 2ull * r.blocks * r.tile_rows * (c.D + 1) * sizeof(float) + r.blocks * sizeof(PagedHead);
  }
  return r;
}

template <typename T, int D, int kRows>
static int launch_rows(const FaPagedParams& p, int blocks, cudaStream_t stream) {
  using Smem = FaPagedSmem<D, kRows>;
  auto kernel = fa_paged_rows_kernel<T, D, kRows>;
  static bool configured[64] = {};
  int dev = 0;
  HB_CUDA_CHECK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(g_paged_mutex);
    if (!configured[dev & 63]) {
      HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem)));
      HB_CUDA_CHECK(cudaFuncSetAttribute(fa_paged_combine_kernel<T, D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      configured[dev & 63] = true;
    }
  }
  HB_CUDA_CHECK(launch_dependent(kernel, blocks, kPagedThreads, sizeof(Smem), stream, 0, p));
  return HB_OK;
}
template <typename T, int D>
static int launch_combine(const FaPagedParams& p, int rows, int blocks, cudaStream_t stream) {
  // parts of an item, where all items are alike
  const long long items = static_cast<long long>(p.c.B) * p.c.Hkv;
  const long long parts = (blocks + items - 1) / items + 1;
  // warps to a row, rows of a block.  us, B1 Hq32 Hkv8 D128 1000 keys (17 parts) with 2 x 8 | 4 x 2 | 8 x 1: 9.1 | 8.6 | 9.1, B3 Hq64 60011 keys (20) 54.4 | 54.0 | 56.5
  const int warps = parts <= 6 ? 1 : parts <= 64 ? 4 : kPagedCombineWarps, rows_here = warps == 1 ? 8 : warps == 4 ? 2 : 1;
  HB_CUDA_CHECK(launch_dependent(fa_paged_combine_kernel<T, D>, blocks * (rows / rows_here), 32 * warps * rows_here, 0, stream, 0, p, rows, warps));
  return HB_OK;
}
template <typename T>
static int launch_rows_of(const FaPagedParams& p, int D, int rows, int blocks, cudaStream_t stream) {
  if (D == 128) return rows == 8 ? launch_rows<T, 128, 8>(p, blocks, stream) : launch_rows<T, 128, 16>(p, blocks, stream);
  return rows == 8 ? launch_rows<T, 64, 8>(p, blocks, stream) : launch_rows<T, 64, 16>(p, blocks, stream);
}
template <typename T>
static int launch_combine_of(const FaPagedParams& p, int D, int rows, int blocks, cudaStream_t stream) {
  return D == 128 ? launch_combine<T, 128>(p, rows, blocks, stream) : launch_combine<T, 64>(p, rows, blocks, stream);
}

template <typename T, int D>
static int launch_tiles(const FaPagedTilesParams& p, unsigned grid, int smem_optin, cudaStream_t stream) {
  using Smem = FaPagedTilesSmem<D>;
  if ((int)sizeof(Smem) > smem_optin)
    return set_error(HB_ERR_UNSUPPORTED, "hb_fa_paged: kernel needs %d bytes of shared memory, device offers %d", (int)sizeof(Smem), smem_optin);
  auto kernel = fa_paged_tiles_kernel<T, D>;
  static bool configured[64] = {};
  int dev = 0;
  HB_CUDA_CHECK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(g_paged_mutex);
    if (!configured[dev & 63]) {
      HB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem)));
      configured[dev & 63] = true;
    }
  }
  HB_CUDA_CHECK(launch_dependent(kernel, grid, kPagedTilesThreads, sizeof(Smem), stream, 0, p));
  return HB_OK;
}
template <typename T>
static int launch_tiles_of(const FaPagedTilesParams& p, int D, unsigned grid, int smem_optin, cudaStream_t stream) {
  return D == 128 ? launch_tiles<T, 128>(p, grid, smem_optin, stream) : launch_tiles<T, 64>(p, grid, smem_optin, stream);
}

}  // namespace hb

extern "C" int hb_fa_paged_workspace(const hb_fa_paged_args* a, uint64_t* bytes) {
  using namespace hb;
  clear_error();
  if (bytes == nullptr) return set_error(HB_ERR_BAD_ARG, "hb_fa_paged_workspace: bytes is NULL");
  *bytes = 0;
  bool empty = false;
  int rc = paged_check("hb_fa_paged_workspace", a, &empty);
  if (rc != HB_OK || empty) return rc;
  DeviceState* st = nullptr;
  rc = get_device_state(&st);
  if (rc != HB_OK) return rc;
  *bytes = paged_route(a, st->sm_count).bytes;
  return HB_OK;
}

extern "C" int hb_fa_paged(const hb_fa_paged_args* a, void* workspace, uint64_t bytes) {
  using namespace hb;
  clear_error();
  bool empty = false;
  int rc = paged_check("hb_fa_paged", a, &empty);
  if (rc != HB_OK || empty) return rc;
  DeviceState* st = nullptr;
  rc = get_device_state(&st);
  if (rc != HB_OK) return rc;
  const PagedRoute route = paged_route(a, st->sm_count);
  if (route.items > 0x7fffffffll / (kPagedBlockRows / 32)) return set_error(HB_ERR_UNSUPPORTED, "hb_fa_paged: more than 2^31 blocks of query rows");
  const uint64_t need = route.bytes;
  if (need > 0 && (workspace == nullptr || bytes < need))
    return set_error(HB_ERR_BAD_ARG, "hb_fa_paged: needs a workspace of %llu bytes, got %llu", (unsigned long long)need,
                     (unsigned long long)(workspace == nullptr ? 0 : bytes));
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return set_error(HB_ERR_ALIGN, "hb_fa_paged: the workspace must be 16-byte aligned");
  const hb_kv_cache& c = a->cache;
  const float scale = a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / sqrtf((float)c.D);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  auto fill = [&](auto& p) {
    p.c = kv_view(c, st);
    p.q = a->q;
    p.o = a->o;
    p.lse = a->lse;
    p.q_st = a->q_stride_t;
    p.q_sh = a->q_stride_h;
    p.o_st = a->o_stride_t;
    p.o_sh = a->o_stride_h;
    p.Hq = a->Hq;
    p.group = a->Hq / c.Hkv;
    p.causal = a->causal ? 1 : 0;
    p.by_group = make_fast_div(p.group);
    p.scale_log2 = scale * 1.4426950408889634f;
  };
  FaPagedParams p;
  const int rows = route.tile_rows, blocks = route.blocks;
  if (route.rows_kernel) {
    fill(p);
    p.row_limit = route.tiles_kernel ? route.row_limit : INT_MAX;
    p.status = st->status_word;
    for (const bool keys : {true, false}) {
      // an axis of one page, head or token may carry any stride
      const uint64_t dims[4] = {(uint64_t)c.D, (uint64_t)c.page_size, (uint64_t)c.Hkv, (uint64_t)std::max(c.num_pages, 1)};
      const int64_t given[3] = {keys ? c.k_stride_s : c.v_stride_s, keys ? c.k_stride_h : c.v_stride_h, keys ? c.k_stride_p : c.v_stride_p};
      uint64_t strides[3];
      for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] > 1 ? (uint64_t)given[i] : (uint64_t)c.D;
      const uint32_t box[4] = {(uint32_t)c.D, (uint32_t)std::min(c.page_size, paged_tile(c.D)), 1, 1};
      rc = encode_tensor_map(keys ? &p.tm_k : &p.tm_v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, keys ? c.k : c.v, dims, strides, box,
                             c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
      if (rc != HB_OK) return rc;
    }
    p.heads = reinterpret_cast<PagedHead*>(static_cast<uint8_t*>(workspace) + route.tiles_bytes);
    p.part_o = reinterpret_cast<float*>(p.heads + blocks);
    p.part_lse = p.part_o + 2ll * blocks * rows * c.D;
    rc = a->dtype == HB_BF16 ? launch_rows_of<__nv_bfloat16>(p, c.D, rows, blocks, stream) : launch_rows_of<__half>(p, c.D, rows, blocks, stream);
    if (rc != HB_OK) return rc;
  }
  FaPagedTilesParams t;
  const int64_t items = route.items;
  if (items > 0) {
    fill(t);
    t.row_limit = route.row_limit;
    t.by_hkv = make_fast_div(c.Hkv);
    t.by_b = make_fast_div(c.B);
    t.status = st->status_word;
    t.splits = route.splits;
    t.parts = static_cast<PagedParts*>(workspace);
    t.part_o = t.splits > 1 ? reinterpret_cast<float*>(t.parts + items) : nullptr;
    t.part_lse = t.splits > 1 ? t.part_o + items * t.splits * kPagedBlockRows * c.D : nullptr;
    const unsigned grid = static_cast<unsigned>(items * t.splits);
    rc = a->dtype == HB_BF16 ? launch_tiles_of<__nv_bfloat16>(t, c.D, grid, st->smem_optin, stream)
                             : launch_tiles_of<__half>(t, c.D, grid, st->smem_optin, stream);
    if (rc != HB_OK) return rc;
  }
  if (route.rows_kernel) {
    rc = a->dtype == HB_BF16 ? launch_combine_of<__nv_bfloat16>(p, c.D, rows, blocks, stream) : launch_combine_of<__half>(p, c.D, rows, blocks, stream);
    if (rc != HB_OK) return rc;
  }
  if (items == 0 || t.splits == 1) return HB_OK;
  const unsigned grid = static_cast<unsigned>(items * (kPagedBlockRows / 32));
  cudaError_t err;
  if (a->dtype == HB_BF16)
    err = c.D == 128 ? launch_dependent(fa_paged_tiles_combine_kernel<__nv_bfloat16, 128>, grid, 256, 0, stream, 0, t)
                     : launch_dependent(fa_paged_tiles_combine_kernel<__nv_bfloat16, 64>, grid, 256, 0, stream, 0, t);
  else
    err = c.D == 128 ? launch_dependent(fa_paged_tiles_combine_kernel<__half, 128>, grid, 256, 0, stream, 0, t)
                     : launch_dependent(fa_paged_tiles_combine_kernel<__half, 64>, grid, 256, 0, stream, 0, t);
  HB_CUDA_CHECK(err);
  return HB_OK;
}
