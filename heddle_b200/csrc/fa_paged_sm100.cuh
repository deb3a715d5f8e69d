// Attention of few query rows over the paged 8-bit cache (hb_fa_paged), sm_100a.
//
//   s_ij = scale (q_i . K_j) kscale[page(j)],   o_i = sum_j softmax(s_i)_j V_j vscale[page(j)],   K, V e4m3 codes
//
// What bounds it is reading the codes once: 2 D bytes a token and KV head, 11 cycles of an SM's share of HBM at D = 128.
// The products are mma.sync m16n8k16 in fp16, which holds every code exactly, and a query too once its row is scaled by a power of two
// (2^-39 of the row's largest element is its last place).  Codes are converted as they come from shared memory, two at an
// instruction; 8-bit products of mma.sync are no way around that: on sm_100 they are converted as well, operand by operand and
// product by product (5.9 cycles of an SM for m16n8k32 against 2.0 for the fp16 product of half that depth).  So the codes are A and the
// few query rows B: S^T = K Q^T (16 keys by 8 rows) and O^T = V^T P^T, and nothing is padded beyond 8 rows.
//
// A warp works through tiles of 32 keys (64 at D = 64) alone, from its own ring in shared memory, filled by TMA copies of a page's tokens (as 16-byte
// asynchronous copies of each lane a tile's loads took 800 of its 3000 cycles).  Keys are numbered within a group of eight so that both readings of a tile (keys
// along their rows, values across them) are free of bank conflicts; P goes from S^T's layout into B's by a transposing move,
// and the pairs of value rows that a lane needs are put together by byte permutations.
// What a row keeps the maximum of is score + log2 vscale, of the keys that it sees, so that P' = 2^8 P vscale, relative to that, is a number of fp16
// whatever the scales are: it is 2^-33 of the row's largest product of weight and value scale at its finest.  The sum of the weights takes
// the scales out again, by powers of two that fp32 holds.  A maximum is adopted when it grew by more than 2^7, as in fa_fwd.
//
// Work: the list of fa_paged_plan.h.  A run may start or end inside an item: such a segment leaves fp32 partial results in the
// workspace, and fa_paged_combine_kernel merges them.
//
// us in a captured graph, both kernels (bytes the call cannot do without): B64 Hq32 Hkv8 D128, one token, 2000 to 4100 keys 69.7 (406 MB, 5.8 TB/s); B3 Hq64
// Hkv8 D128, 30 to 60 thousand keys 52.8 (5.3 TB/s); B24 Hq32 Hkv8 D128, four tokens, 1500 to 3000 keys 34.4 (3.3); B40 Hq12 Hkv12 D64 26.4 (3.1); B1, 1000 keys 8.6.
// About 10 us of each are the start (list, first pages), the meeting of the warps and the merge; the loop itself reads 5 to 6 TB/s.
#pragma once

#include "fa_paged_plan.h"
#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace hb {

constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedMaxRows = 16;
constexpr uint32_t kRolePagedRows = 14;
constexpr float kPagedBits = 8.f, kPagedGrowth = 7.f;  // P' = 2^(kPagedBits + score - m): at most 2^15, since m is adopted behind kPagedGrowth

struct alignas(16) PagedHead {  // of an item in parts: where its parts lie (one a run; written by the run that starts the item)
  int last;         // run of its last part, -1: this run starts no item in parts
  int slot;         // of its first part
  int h, row0;      // KV head, first row of the row tile
  int start, rows;  // of the sequence: its first row of the call, its query rows in a KV head
  int pad[2];
};

struct alignas(64) FaPagedParams {
  CUtensorMap tm_k, tm_v;  // pages as [page][head][token][D], boxes of a tile's tokens (of a page's, where it has fewer)
  KvView c;
  const void* q;
  void* o;
  float* lse;
  long long q_st, q_sh, o_st, o_sh;
  int Hq, group, causal;
  int row_limit;    // sequences with more query rows a KV head are not this kernel's
  FastDiv by_group;
  float scale_log2;
  uint32_t* status;
  float* part_o;    // [2 * blocks][rows][D], O / l
  float* part_lse;  // [2 * blocks][rows], base 2
  PagedHead* heads; // [blocks]
};

// Blocks an SM holds: what bounds a warp is the latency of its own instructions (four cycles and a half each with two warps to a
// scheduler), so registers and the ring are cut to fit as many warps as do not spill.
template <int D, int kRows>
constexpr int paged_blocks_per_sm = kRows == 8 || D == 64 ? 3 : 2;

template <int D, int kRows>
struct FaPagedSmem {
  static constexpr int kTile = paged_tile(D), kGroups = kTile / 16;
  static constexpr int kTileBytes = kTile * D;  // of keys, and of values
  static constexpr int kStages = paged_blocks_per_sm<D, kRows> == 3 ? 2 : 3;
  static constexpr int kFrags = kRows / 8 * (D / 16);  // accumulator tiles of O^T
  alignas(1024) uint8_t ring[kPagedWarps][kStages][2 * kTileBytes];
  float4 o[kPagedWarps / 2][kFrags][32];   // a warp's accumulators, as its lanes hold them ...
  float ml[kPagedWarps / 2][2][kRows];     // ... and its maxima and sums
  alignas(16) float scales[kPagedWarps][kStages][2 * kGroups];  // of keys, of values of each 16 keys; 0: behind the sequence, or no page of the cache's
  uint64_t full[kPagedWarps][kStages];
  long long sums[kPagedWarps];
  long long found_at;
  int found;
  uint32_t abort_flag;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The codes of a word's lower and upper half as fp16 pairs.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// An 8 x 8 matrix of 16-bit numbers, a row's pair in each lane, transposed.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(addr) : "memory");
  return w;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 w;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(addr) : "memory");
  return w;
}
// four bytes, or zeros where there is nothing to copy
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
// sixteen bytes, or zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A place in the list of key tiles.
struct PagedCursor {
  int b;
  KvSeq s;
  int tiles, row_tiles;  // of the sequence's items
  int h, rt;
  int j;                 // key tile
};
// The sequence's part of the list: 0 where it has no rows, or too many for this kernel.
__device__ __forceinline__ long long paged_list(const FaPagedParams& p, const KvSeq& s, int rows, int tile, int& tiles, int& row_tiles) {
  tiles = paged_tiles(s.len, tile);
  row_tiles = static_cast<long long>(s.n) * p.group <= p.row_limit ? paged_row_tiles(s.n, p.group, rows) : 0;
  return static_cast<long long>(paged_places(tiles)) * row_tiles * p.c.Hkv;
}
__device__ __forceinline__ void paged_enter(const FaPagedParams& p, PagedCursor& at, int rows, int tile) {
  at.s = kv_seq(p.c, at.b);
  (void)paged_list(p, at.s, rows, tile, at.tiles, at.row_tiles);
}
// To the first tile of the next item; only where the list has one.
__device__ __forceinline__ void paged_next_item(const FaPagedParams& p, PagedCursor& at, int rows, int tile) {
  if (++at.rt < at.row_tiles) return;
  at.rt = 0;
  if (++at.h < p.c.Hkv) return;
  at.h = 0;
  do {
    if (++at.b >= p.c.B) return;
    paged_enter(p, at, rows, tile);
  } while (at.row_tiles == 0);
}

template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kPagedThreads, (paged_blocks_per_sm<D, kRows>)) fa_paged_rows_kernel(const __grid_constant__ FaPagedParams p) {
  using Smem = FaPagedSmem<D, kRows>;
  constexpr int kTile = Smem::kTile, kGroups = Smem::kGroups;
  constexpr int kSteps = D / 16;  // products along head_dim
  constexpr int kDims = D / 16;   // accumulator tiles of O^T along head_dim
  constexpr int kN = kRows / 8;   // tiles of query rows
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const KvView& kv = p.c;
  AbortCtx ctx{&sm.abort_flag, p.status};
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    for (int w = 0; w < kPagedWarps; ++w)
      for (int i = 0; i < Smem::kStages; ++i) mbar_init(&sm.full[w][i], 1);
    fence_mbar_init();
    if ((smem_u32(smem_raw) & 1023u) != 0u) raise_abort(ctx, kStatusSmemMisaligned);
    prefetch_tensormap(&p.tm_k);
    prefetch_tensormap(&p.tm_v);
  }
  grid_wait();

  // ---- this block's run of the list: the sequences' parts are added up in rounds of a block's threads
  long long total = 0, own = 0, upto = 0;  // own: of the last round
  bool descends = false;                   // see kv_descends
  for (int b0 = 0; b0 < kv.B; b0 += kPagedThreads) {
    const int b = b0 + threadIdx.x;
    int tiles, row_tiles;
    own = upto = b < kv.B ? paged_list(p, kv_seq(kv, b), kRows, kTile, tiles, row_tiles) : 0;
    const bool down = kv.starts != nullptr && b < kv.B && kv_start(kv, b) > kv_start(kv, b + 1);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (b0 > 0) __syncthreads();
    if (lane == 31) sm.sums[warp] = upto;
    if (__syncthreads_or(down)) descends = true;
    upto += total;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      if (w < warp) upto += sm.sums[w];
      total += sm.sums[w];
    }
  }
  const int run = blockIdx.x;
  if (threadIdx.x == kPagedThreads - 32) p.heads[run].last = -1;  // the thread that may write another one
  if (run == 0) {
    for (int b = threadIdx.x; b < kv.B; b += kPagedThreads) {
      const uint32_t f = kv_seq_faults(kv, b);
      if (f != 0) kv_report(kv, f);
    }
  }
  const int runs = paged_runs(total, gridDim.x);
  if (total == 0 || run >= runs || descends) return;
  const long long begin = paged_begin(total, runs, run), end = paged_begin(total, runs, run + 1);
  if (kv.B <= kPagedThreads) {
    if (upto > begin && upto - own <= begin) {
      sm.found = threadIdx.x;
      sm.found_at = upto - own;
    }
  } else {
    long long before = 0;  // of the sequences in front of this round's
    for (int b0 = 0; b0 < kv.B && before <= begin; b0 += kPagedThreads) {
      const int b = b0 + threadIdx.x;
      int tiles, row_tiles;
      own = upto = b < kv.B ? paged_list(p, kv_seq(kv, b), kRows, kTile, tiles, row_tiles) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      __syncthreads();
      if (lane == 31) sm.sums[warp] = upto;
      __syncthreads();
      upto += before;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        if (w < warp) upto += sm.sums[w];
        before += sm.sums[w];
      }
      if (upto > begin && upto - own <= begin) {
        sm.found = b;
        sm.found_at = upto - own;
      }
    }
  }
  __syncthreads();

  PagedCursor seg;  // the segment's item and first tile
  seg.b = sm.found;
  paged_enter(p, seg, kRows, kTile);
  long long t = begin;  // place of the segment's first tile in the list
  {
    const int places = paged_places(seg.tiles);
    const long long in = begin - sm.found_at, item = paged_div(in, places);
    const int at = static_cast<int>(in - item * places);
    seg.j = max(at - kPagedItemCost, 0);
    t += max(kPagedItemCost - at, 0);
    seg.h = static_cast<int>(paged_div(item, seg.row_tiles));
    seg.rt = static_cast<int>(item - static_cast<long long>(seg.h) * seg.row_tiles);
  }
  if (t >= end) return;  // a short run, all of it in front of an item's tiles

  // ---- the queries of a segment, as they come: columns 16 (c + 4 hh) .. + 15 of row g of each row tile
  uint4 q_raw[kN][D / 64][2];
  auto fetch_q = [&](const PagedCursor& at) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int row = at.rt * kRows + 8 * n + g;
      const bool live = row < at.s.n * p.group;
      const int tok = live ? fast_div(row, p.by_group) : 0, head = live ? row - tok * p.group : 0;
      const T* src = static_cast<const T*>(p.q) + (at.s.start + tok) * p.q_st + (at.h * p.group + head) * p.q_sh + 16 * c;
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) {
#pragma unroll
        for (int e = 0; e < 2; ++e) q_raw[n][hh][e] = live ? *reinterpret_cast<const uint4*>(src + 64 * hh + 8 * e) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  // A segment of one tile is its warp's alone, which stores the rows by itself: short items go to the warps in turn, and nobody waits.  us
  // without | with: B128 Hq16 D128, 20 keys 18.6 | 11.4; B100 Hq32 Hkv8 D128, four tokens on themselves 18.4 | 9.6.
  auto alone = [&](const PagedCursor& at, long long place) -> bool { return end - place == 1 || at.tiles - at.j == 1; };
  int turn = 0;  // tiles of the run in front of the segment, modulo the warps
  bool solo = alone(seg, t), mine = !solo || warp == 0;
  if (mine) fetch_q(seg);  // in front of the tiles, which the memory takes its time over

  // ---- loads: the warp's next tile, while the ids of the pages of the one after are on their way
  PagedCursor ld = seg;
  long long ld_left = end - t;  // places of the run from ld's tile on; the warp's tiles are every fourth
  auto skip = [&](int tiles) {
    ld.j += tiles;
    ld_left -= tiles;
    while (ld.j >= ld.tiles && ld_left > kPagedItemCost) {
      ld.j -= ld.tiles;
      ld_left -= kPagedItemCost;
      paged_next_item(p, ld, kRows, kTile);
    }
    if (ld.j >= ld.tiles) ld_left = 0;
  };
  // the page of keys 16 (lane % kGroups) .. + 15 of the tile, as the table has it (-1: behind the sequence); looked at when it is used: a
  // warp stops where it looks at what has not come yet
  const int group0 = 16 * (lane & (kGroups - 1));
  auto page_of = [&]() -> int {
    const int tok = ld.j * kTile + group0;
    return tok < ld.s.len ? kv.table[ld.b * kv.table_stride + (tok >> kv.page_shift)] : -1;
  };
  int page = -1;
  skip(warp);
  if (ld_left > 0) page = page_of();
  uint32_t ld_stage = 0;
  const int no_page = max(kv.num_pages, 1);  // the first coordinate outside of the cache: the copy writes zeros
  const bool copies = lane < kGroups && (group0 & (min(1 << kv.page_shift, kTile) - 1)) == 0;  // the lane's keys begin a copy
  auto load = [&]() {                  // one tile, or nothing behind the run's end: a group of copies of scales either way
    if (ld_left > 0) {
      const int tok = ld.j * kTile + group0, h = ld.h, len = ld.s.len;
      const int id = static_cast<unsigned>(page) < static_cast<unsigned>(kv.num_pages) ? page : -1;
      skip(kPagedWarps);
      if (ld_left > 0) page = page_of();
      uint64_t* bar = &sm.full[warp][ld_stage];
      if (lane == 0) mbar_arrive_expect_tx(bar, 2 * Smem::kTileBytes);
      __syncwarp();
      if (copies) {
        uint8_t* dst = sm.ring[warp][ld_stage] + group0 * D;
        const int at = tok & ((1 << kv.page_shift) - 1), coord = id < 0 ? no_page : id;
        tma_load_4d(dst, &p.tm_k, bar, 0, at, h, coord);
        tma_load_4d(dst + Smem::kTileBytes, &p.tm_v, bar, 0, at, h, coord);
      }
      if (lane < 2 * kGroups) {
        if (id < 0 && tok < len) kv_report(kv, HB_CACHE_BAD_PAGE);
        const float* src = (lane >= kGroups ? kv.v_scale : kv.k_scale) + (id >= 0 ? static_cast<long long>(id) * kv.Hkv + h : 0);
        cp_async4(smem_u32(&sm.scales[warp][ld_stage][lane]), src, id >= 0);
      }
      if (++ld_stage == Smem::kStages) ld_stage = 0;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < Smem::kStages - 1; ++i) load();

  // ---- what the lane reads of a tile: of keys, row g ^ 4 (g & 1) of a group of eight, chunks c (and c + 4); of values, rows 2 c and
  // (2 c + 1) ^ 4, D / 8 columns
  uint32_t k_at[D / 64], v_at[2];
  {
    const int key = g ^ ((g & 1) << 2);
#pragma unroll
    for (int hh = 0; hh < D / 64; ++hh) k_at[hh] = key * D + (D == 128 ? (c + 4 * hh) ^ key : c ^ (key >> 1)) * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (2 * c + i) ^ (i << 2);
      v_at[i] = row * D + (D == 128 ? (g ^ row) * 16 : ((g >> 1) ^ (row >> 1)) * 16 + (g & 1) * 8);
    }
  }

  // ---- segments
  uint32_t stage = 0, phase = 0;
  bool alive = true;  // until a wait gives up: then the block's barriers are all that is left to do
  bool first = true;
  while (t < end) {
    const long long left = end - t;
    const int j0 = seg.j, j1 = left < seg.tiles - j0 ? j0 + static_cast<int>(left) : seg.tiles;
    const int rows = seg.s.n * p.group, row0 = seg.rt * kRows;
    const bool whole = j0 == 0 && j1 == seg.tiles;
    const int slot = 2 * run + (first ? 0 : 1);
    const long long last = t + (seg.tiles - 1 - j0);  // place of the item's last tile
    const bool more = last + kPagedItemCost + 1 < end;
    const int next_turn = (turn + (j1 - j0)) & (kPagedWarps - 1);
    if (warp == kPagedWarps - 1 && lane == 0 && j0 == 0 && !whole) {
      PagedHead hd;
      hd.last = paged_run_of(total, runs, last);
      hd.slot = slot;
      hd.h = seg.h;
      hd.row0 = row0;
      hd.start = seg.s.start;
      hd.rows = rows;
      p.heads[run] = hd;
    }
    if (!mine) {
      if (!more) break;
      paged_next_item(p, seg, kRows, kTile);
      seg.j = 0;
      t = last + kPagedItemCost + 1;
      first = false;
      turn = next_turn;
      solo = alone(seg, t);
      mine = !solo || warp == turn;
      if (mine) fetch_q(seg);
      continue;
    }

    // B of S^T: the lane has columns 16 (c + 4 hh) .. + 15 of row g of each tile, scaled by 2^up, which takes the row's largest element
    // into [2^14, 2^15).  What it does with scores needs rows 2 c and 2 c + 1.
    uint32_t qf[kN][kSteps][2];
    float factor[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float x[D / 64][16];
      float top = 0.f;
      bool finite = true;
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) {
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          const uint4 w = q_raw[n][hh][e >> 3];
          Pack2<T>::unpack(w.x, x[hh][e], x[hh][e + 1]);
          Pack2<T>::unpack(w.y, x[hh][e + 2], x[hh][e + 3]);
          Pack2<T>::unpack(w.z, x[hh][e + 4], x[hh][e + 5]);
          Pack2<T>::unpack(w.w, x[hh][e + 6], x[hh][e + 7]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          top = fmaxf(top, fabsf(x[hh][e]));
          finite = finite && fabsf(x[hh][e]) <= 3.402823466e38f;
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int up = 0;
      if (top > 0.f && top <= 3.402823466e38f) up = min(14 - ((__float_as_int(top) >> 23) - 127), 120);
      // a row that holds an infinity or NaN is NaN: its scores are, those of keys that it sees
      const unsigned votes = __ballot_sync(0xffffffffu, finite);
      const float mul = ((votes >> (lane & ~3)) & 15u) == 15u ? __int_as_float((up + 127) << 23) : __int_as_float(0x7fc00000);
      const float f = p.scale_log2 * __int_as_float((127 - up) << 23);
#pragma unroll
      for (int e = 0; e < 2; ++e) factor[n][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * c + e));
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[n][4 * hh + (e >> 1)][e & 1] = Pack2<__half>::pack(x[hh][2 * e] * mul, x[hh][2 * e + 1] * mul);
      }
    }
    // keys that every live row sees: the first row's token sees least
    const int least = p.causal ? min(seg.s.len, seg.s.pos0() + fast_div(row0, p.by_group) + 1) : seg.s.len;

    float o[kN][kDims][4];
    // value scales are relative to `base`, the first tile's largest; m: the largest score + log2 vscale / base; O is in 2^(m - kPagedBits) base, l in
    // 2^(m - kPagedBits)
    float m[kN][2], l[kN][2];
    int base = 0;  // bits; 0: no tile yet
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    for (int j = j0 + ((warp - turn) & (kPagedWarps - 1)); j < j1; j += kPagedWarps) {
      cp_async_wait<Smem::kStages - 2>();
      alive = alive && mbar_wait_warp(&sm.full[warp][stage], phase, ctx, kRolePagedRows);
      if (!alive) break;
      __syncwarp();  // every lane's scales are there, and every lane is done with the tile before: its stage is free
      load();
      const uint32_t tile = smem_u32(sm.ring[warp][stage]);
      float ks[kGroups], vs[kGroups];  // a group: 16 keys
#pragma unroll
      for (int t = 0; t < 2 * kGroups; t += 4) {
        const float4 y = *reinterpret_cast<const float4*>(&sm.scales[warp][stage][t]);
        const float z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) (t + e < kGroups ? ks[(t + e) % kGroups] : vs[(t + e) % kGroups]) = z[e];
      }

      // scores of the tile's keys: row r of group t is key 16 t + (r ^ 4 (r & 1)); the lane has rows g and g + 8, columns 2 c and 2 c + 1
      float x[kN][kGroups][4];
#pragma unroll
      for (int t = 0; t < kGroups; ++t) {
#pragma unroll
        for (int n = 0; n < kN; ++n) x[n][t][0] = x[n][t][1] = x[n][t][2] = x[n][t][3] = 0.f;
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh) {
          const uint4 ka = lds128(tile + k_at[hh] + 16 * t * D), kb = lds128(tile + k_at[hh] + (16 * t + 8) * D);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            codes_f16(wa[w], a0, a2);
            codes_f16(wb[w], a1, a3);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_f16(x[n][t], a0, a1, a2, a3, qf[n][4 * hh + w][0], qf[n][4 * hh + w][1]);
          }
        }
      }
      // keys that a row does not see, or that are not there
      bool there = true, valued = true;
      int v_top = 0;
#pragma unroll
      for (int t = 0; t < kGroups; ++t) {
        there = there && ks[t] != 0.f;
        valued = valued && vs[t] != 0.f;
        v_top = max(v_top, ks[t] != 0.f ? __float_as_int(vs[t]) : 0);
      }
      if (base == 0) base = v_top;
      if ((j + 1) * kTile > least || !there) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = row0 + 8 * n + 2 * c + e;
            const int limit = r >= rows ? 0 : p.causal ? min(seg.s.len, seg.s.pos0() + fast_div(r, p.by_group) + 1) : seg.s.len;
            const int key = j * kTile + (g ^ ((g & 1) << 2));
#pragma unroll
            for (int t = 0; t < kGroups; ++t) {
              if (ks[t] == 0.f || key + 16 * t >= limit) x[n][t][e] = -INFINITY;
              if (ks[t] == 0.f || key + 16 * t + 8 >= limit) x[n][t][2 + e] = -INFINITY;
            }
          }
        }
      }
      bool moved = false;
      float v_log[kGroups], v_inv[kGroups];  // log2 vscale / base and its inverse; where the scale is 0, as if it were base, and the values are 0
#pragma unroll
      for (int t = 0; t < kGroups; ++t) {
        const int to = vs[t] != 0.f ? min(max(__float_as_int(vs[t]) - base, -(126 << 23)), 126 << 23) : 0;
        v_log[t] = static_cast<float>(to >> 23);
        v_inv[t] = __int_as_float((127 << 23) - to);
      }
      float alpha[kN][2];
      uint32_t pb[kN][kGroups][2];  // P' as B of O^T
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // not 0 (a page without a scale, or less than fp32 holds): -inf has to stay it
          float f[kGroups], top = -INFINITY;
#pragma unroll
          for (int t = 0; t < kGroups; ++t) {
            f[t] = factor[n][e] * ks[t];
            f[t] = f[t] == 0.f ? 1.17549435e-38f : f[t];
            top = fmaxf(top, fmaf(fmaxf(x[n][t][e], x[n][t][2 + e]), f[t], v_log[t]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const bool adopt = top > m[n][e] + kPagedGrowth;  // of -inf: any maximum
          alpha[n][e] = adopt ? fast_exp2(m[n][e] - top) : 1.f;
          moved = moved || adopt;
          m[n][e] = adopt ? top : m[n][e];
          // the 2^kPagedBits go in here, in front of the rounding to fp16: its numbers below 2^-14 lose bits, those below 2^-25 are 0
          const float off = kPagedBits - (m[n][e] == -INFINITY ? 0.f : m[n][e]);
          float sum = 0.f;
#pragma unroll
          for (int t = 0; t < kGroups; ++t) {
            const float off_t = off + v_log[t];
            x[n][t][e] = fast_exp2(fmaf(x[n][t][e], f[t], off_t));
            x[n][t][2 + e] = fast_exp2(fmaf(x[n][t][2 + e], f[t], off_t));
            sum = fmaf(x[n][t][e] + x[n][t][2 + e], v_inv[t], sum);
          }
          l[n][e] = fmaf(l[n][e], alpha[n][e], sum);
        }
#pragma unroll
        for (int t = 0; t < kGroups; ++t) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const __half2 y = __floats2half2_rn(x[n][t][2 * h], x[n][t][2 * h + 1]);
            pb[n][t][h] = movmatrix(*reinterpret_cast<const uint32_t*>(&y));
          }
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const float f0 = alpha[n][0], f1 = alpha[n][1];
#pragma unroll
          for (int i = 0; i < kDims; ++i) {
            o[n][i][0] *= f0;
            o[n][i][1] *= f1;
            o[n][i][2] *= f0;
            o[n][i][3] *= f1;
          }
        }
      }
      // O^T += V^T P'^T: of group t the lane has value rows 2 c, (2 c + 1) ^ 4 and those plus 8, columns D / 8 from D / 8 g on: rows g and
      // g + 8 of tile i are columns 2 i and 2 i + 1 of them
#pragma unroll
      for (int t = 0; t < kGroups; ++t) {
        constexpr int kWords = D / 32;  // of 4 columns
        uint32_t vw[4][kWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at = tile + Smem::kTileBytes + (16 * t + 8 * (i >> 1)) * D + v_at[i & 1];
          if constexpr (D == 128) {
            const uint4 w = lds128(at);
            vw[i][0] = w.x;
            vw[i][1] = w.y;
            vw[i][2] = w.z;
            vw[i][3] = w.w;
          } else {
            const uint2 w = lds64(at);
            vw[i][0] = w.x;
            vw[i][1] = w.y;
          }
        }
        // what a page holds behind the sequence is loaded with it; as numbers it may be anything, and 0 times it has to be 0
        if ((j + 1) * kTile > seg.s.len || !valued) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = j * kTile + 16 * t + 8 * (i >> 1) + ((2 * c + (i & 1)) ^ ((i & 1) << 2));
#pragma unroll
            for (int w = 0; w < kWords; ++w) vw[i][w] = key < seg.s.len && sm.scales[warp][stage][kGroups + t] != 0.f ? vw[i][w] : 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t pick = half == 0 ? 0x5140u : 0x7362u;
            uint32_t a0, a1, a2, a3;
            codes_f16(__byte_perm(vw[0][w], vw[1][w], pick), a0, a1);
            codes_f16(__byte_perm(vw[2][w], vw[3][w], pick), a2, a3);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_f16(o[n][2 * w + half], a0, a1, a2, a3, pb[n][t][0], pb[n][t][1]);
          }
        }
      }
      if (++stage == Smem::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    PagedCursor next = seg;
    bool next_solo = false, next_mine = false;
    if (more) {
      paged_next_item(p, next, kRows, kTile);
      next.j = 0;
      next_solo = alone(next, last + kPagedItemCost + 1);
      next_mine = !next_solo || warp == next_turn;
      if (next_mine) fetch_q(next);
    }

    // ---- the warps' results meet: 2 and 3 hand theirs to 0 and 1, 1 to 0, which stores the rows
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
        l[n][e] *= 1.f / 256.f;
      }
    }
    const float unit = __int_as_float(base) * (1.f / 256.f);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] *= unit;
      }
    }
    auto give = [&](int slot) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < kDims; ++i) sm.o[slot][n * kDims + i][lane] = make_float4(o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
        if (g == 0) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sm.ml[slot][0][8 * n + 2 * c + e] = m[n][e];
            sm.ml[slot][1][8 * n + 2 * c + e] = l[n][e];
          }
        }
      }
    };
    auto take = [&](int slot) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float w0[2], w1[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float other = sm.ml[slot][0][8 * n + 2 * c + e], top = fmaxf(m[n][e], other), safe = top == -INFINITY ? 0.f : top;
          w0[e] = fast_exp2(m[n][e] - safe);
          w1[e] = fast_exp2(other - safe);
          l[n][e] = w0[e] * l[n][e] + w1[e] * sm.ml[slot][1][8 * n + 2 * c + e];
          m[n][e] = top;
        }
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
          const float4 y = sm.o[slot][n * kDims + i][lane];
          o[n][i][0] = w0[0] * o[n][i][0] + w1[0] * y.x;
          o[n][i][1] = w0[1] * o[n][i][1] + w1[1] * y.y;
          o[n][i][2] = w0[0] * o[n][i][2] + w1[0] * y.z;
          o[n][i][3] = w0[1] * o[n][i][3] + w1[1] * y.w;
        }
      }
    };
    if (!solo) {
      if (warp >= 2) give(warp - 2);
      __syncthreads();
      if (warp < 2) take(warp);
      if (warp == 1) {
        __syncwarp();
        give(1);
      }
      __syncthreads();
      if (warp == 0) take(1);
    }
    if (solo || warp == 0) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * n + 2 * c + e, row = row0 + r;
          if (row >= rows) continue;
          const float sum = l[n][e], inv = sum != 0.f ? 1.f / sum : 0.f;  // a row without keys is 0, one with a NaN is NaN
          const float lse2 = sum != 0.f ? (m[n][e] == -INFINITY ? 0.f : m[n][e]) + fast_log2(sum) : -INFINITY;
          if (whole) {
            const int tok = fast_div(row, p.by_group), head = seg.h * p.group + row - tok * p.group;
            T* dst = static_cast<T*>(p.o) + (seg.s.start + tok) * p.o_st + head * p.o_sh + (D / 8) * g;
#pragma unroll
            for (int i = 0; i < kDims; i += 4) {  // 8 columns; rows g, g + 8 of tile i are columns 2 i, 2 i + 1
              uint4 y;
              y.x = Pack2<T>::pack(o[n][i][e] * inv, o[n][i][2 + e] * inv);
              y.y = Pack2<T>::pack(o[n][i + 1][e] * inv, o[n][i + 1][2 + e] * inv);
              y.z = Pack2<T>::pack(o[n][i + 2][e] * inv, o[n][i + 2][2 + e] * inv);
              y.w = Pack2<T>::pack(o[n][i + 3][e] * inv, o[n][i + 3][2 + e] * inv);
              *reinterpret_cast<uint4*>(dst + 2 * i) = y;
            }
            if (g == 0 && p.lse != nullptr) p.lse[static_cast<long long>(seg.s.start + tok) * p.Hq + head] = lse2 * 0.6931471805599453f;
          } else {
            float* dst = p.part_o + (static_cast<long long>(slot) * kRows + r) * D + (D / 8) * g;
#pragma unroll
            for (int i = 0; i < kDims; i += 2)
              *reinterpret_cast<float4*>(dst + 2 * i) =
                  make_float4(o[n][i][e] * inv, o[n][i][2 + e] * inv, o[n][i + 1][e] * inv, o[n][i + 1][2 + e] * inv);
            if (g == 0) p.part_lse[static_cast<long long>(slot) * kRows + r] = lse2;
          }
        }
      }
    }
    if (!solo) __syncthreads();
    turn = next_turn;
    if (!more) break;
    t = last + kPagedItemCost + 1;
    first = false;
    seg = next;
    solo = next_solo;
    mine = next_mine;
  }
  cp_async_wait<0>();
  if (!alive && lane == 0) {  // copies of this warp may be on their way into its ring: give them a while
    for (int i = 0; i < Smem::kStages; ++i)
      for (int spin = 0; spin < 4096 && !mbar_try_wait(&sm.full[warp][i], static_cast<uint32_t>(i) >= stage ? phase : phase ^ 1u); ++spin) {}
  }
  grid_launch_dependents();
}

// Merges the parts of the items that are in any: a block has some rows of one run's head, `warps` warps deal a row's parts out
// between them, a lane has D / 32 columns; weights 2^(lse - max).  What it costs is its chain of loads (head, parts) and the blocks
// that find nothing to do: a block for every row was 3552 of them for 24 items in 18 parts each (B3 Hq64 Hkv8 60011 keys).
constexpr int kPagedCombineWarps = 16;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kPagedCombineWarps) fa_paged_combine_kernel(const __grid_constant__ FaPagedParams p, int kRows, int warps) {
  grid_launch_dependents();
  grid_wait();
  constexpr int kCols = D / 32, kAhead = 4;
  const int rows_here = (blockDim.x >> 5) / warps, blocks_of_run = kRows / rows_here;
  const int run = blockIdx.x / blocks_of_run;
  const PagedHead hd = p.heads[run];
  if (hd.last < 0) return;
  const int warp = uniform_warp(), lane = threadIdx.x & 31, part0 = warp % warps;
  const int r = (blockIdx.x - run * blocks_of_run) * rows_here + warp / warps, row = hd.row0 + r;
  const bool live = row < hd.rows;
  const int parts = live ? hd.last - run + 1 : 0;
  auto at = [&](int part) -> long long { return static_cast<long long>(part == 0 ? hd.slot : 2 * (run + part)) * kRows + r; };
  auto values = [&](int part, float (&x)[kCols]) {
    const float* src = p.part_o + at(part) * D + lane * kCols;
    if constexpr (kCols == 4) {
      const float4 y = *reinterpret_cast<const float4*>(src);
      x[0] = y.x;
      x[1] = y.y;
      x[2] = y.z;
      x[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(src);
      x[0] = y.x;
      x[1] = y.y;
    }
  };
  float ahead[kAhead][kCols];  // the first parts' values are on their way with the weights
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (part0 + i * warps < parts) values(part0 + i * warps, ahead[i]);
  float top = -INFINITY;
  for (int part = lane; part < parts; part += 32) top = fmaxf(top, p.part_lse[at(part)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;
  float acc[kCols] = {}, sum = 0.f;
  for (int part = part0; part < parts; part += kAhead * warps) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int mine = part + i * warps;
      if (mine >= parts) continue;
      const float wt = fast_exp2(p.part_lse[at(mine)] - top);
      sum += wt;
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] = fmaf(wt, ahead[i][e], acc[e]);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (part + (kAhead + i) * warps < parts) values(part + (kAhead + i) * warps, ahead[i]);
  }
  if (warps > 1) {
    __shared__ float s_acc[kPagedCombineWarps][D], s_sum[kPagedCombineWarps];
#pragma unroll
    for (int e = 0; e < kCols; ++e) s_acc[warp][lane * kCols + e] = acc[e];
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (part0 != 0) return;
    for (int k = 1; k < warps; ++k) {
      sum += s_sum[warp + k];
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] += s_acc[warp + k][lane * kCols + e];
    }
  }
  if (!live) return;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  uint32_t packed[kCols / 2];
#pragma unroll
  for (int e = 0; e < kCols; e += 2) packed[e / 2] = Pack2<T>::pack(acc[e] * inv, acc[e + 1] * inv);
  const int tok = fast_div(row, p.by_group), head = hd.h * p.group + row - tok * p.group;
  T* dst = static_cast<T*>(p.o) + (hd.start + tok) * p.o_st + head * p.o_sh + lane * kCols;
  if constexpr (kCols == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  else *reinterpret_cast<uint32_t*>(dst) = packed[0];
  if (lane == 0 && p.lse != nullptr)
    p.lse[static_cast<long long>(hd.start + tok) * p.Hq + head] = (sum != 0.f ? top + fast_log2(sum) : -INFINITY) * 0.6931471805599453f;
}

}  // namespace hb
