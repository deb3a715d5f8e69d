// Attention of few query rows over the paged 8-bit cache (hb_fa_paged), sm_100a.
//
//   s_ij = scale (q_i . K_j) kscale[page(j)],   o_i = sum_j softmax(s_i)_j V_j vscale[page(j)],   K, V e4m3 codes
//
// What bounds it is reading the codes once: 2 D bytes a token and KV head, 11 cycles of an SM's share of HBM at D = 128.  Turning the
// codes over into 16 bits alone would take half of its issue slots, so they go into the tensor cores as they are, and the
// 16-bit operands come to them: a bf16 number has 8 significant bits, an e4m3 one 4, so q (scaled by a power of two that takes
// its row's largest element near 448) is the sum of two e4m3 numbers exactly, three in fp16; P (times 256) is the sum of two to 8 bits.
// mma.sync m16n8k32 on e4m3 adds in full fp32 here (sums of 2^14 and 2^-9 come out exact) and takes 1.07 cycles of an SM, four times
// the multiplications that the 16-bit form does.  With up to 8 rows (kRows) the 16 rows of A are the first parts over the second,
// with up to 16 every part is a product of its own.
//
// A warp works through tiles of 32 keys alone, from its own ring in shared memory, filled by 16-byte asynchronous copies, which
// leave out (as zeros) what lies behind the sequence.  Tokens are numbered within a group of eight so that the score that a lane
// holds is the P that it needs, and both readings of a tile (keys along their rows, values across them) are free of
// bank conflicts.  The four byte columns that a lane has of four value rows are turned over in registers by eight byte permutations.
//
// Work: the list of fa_paged_plan.h.  A run may start or end inside an item: such a segment leaves fp32 partial results in the
// workspace, and fa_paged_combine_kernel merges them.
#pragma once

#include "fa_paged_plan.h"
#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace hb {

constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedMaxRows = 16;

struct PagedHead {  // of an item in parts: where its parts lie (one a run; written by the run that starts the item)
  int b, h, rt;
  int last;  // run of its last part, -1: this run starts no item in parts
  int slot;  // of its first part
  int pad[3];
};

struct FaPagedParams {
  KvView c;
  const void* q;
  void* o;
  float* lse;
  long long q_st, q_sh, o_st, o_sh;
  int Hq, group, causal;
  int row_limit;    // sequences with more query rows a KV head are not this kernel's
  FastDiv by_group;
  float scale_log2;
  float* part_o;    // [2 * blocks][rows][D], O / l
  float* part_lse;  // [2 * blocks][rows], base 2
  PagedHead* heads; // [blocks]
};

template <int D, int kRows>
struct FaPagedSmem {
  static constexpr int kTileBytes = kPagedTile * D;  // of keys, and of values
  static constexpr int kStages = D == 128 ? (kRows == 8 ? 3 : 2) : (kRows == 8 ? 6 : 4);
  alignas(128) uint8_t ring[kPagedWarps][kStages][2 * kTileBytes];
  float o[kPagedWarps][kRows][D];
  float ml[kPagedWarps][2][kRows];
  float scales[kPagedWarps][kStages][4];  // keys, values of the tile's two halves; 0: a page that the cache does not have
  long long sums[kPagedWarps];
  long long found_at;
  int found;
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two numbers rounded to e4m3 (lo in the lower byte) and what is left of them.
__device__ __forceinline__ uint32_t e4m3_part(float& lo, float& hi) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  lo -= f.x;
  hi -= f.y;
  return c;
}
__device__ __forceinline__ uint32_t e4m3_last(float lo, float hi) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
  return c;
}
__device__ __forceinline__ uint32_t e4m3_part4(float (&x)[4]) {
  const uint32_t a = e4m3_part(x[0], x[1]);
  return a | (e4m3_part(x[2], x[3]) << 16);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
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
__device__ __forceinline__ long long paged_list(const FaPagedParams& p, const KvSeq& s, int rows, int& tiles, int& row_tiles) {
  tiles = paged_tiles(s.len);
  row_tiles = static_cast<long long>(s.n) * p.group <= p.row_limit ? paged_row_tiles(s.n, p.group, rows) : 0;
  return static_cast<long long>(tiles) * row_tiles * p.c.Hkv;
}
__device__ __forceinline__ void paged_enter(const FaPagedParams& p, PagedCursor& at, int rows) {
  at.s = kv_seq(p.c, at.b);
  (void)paged_list(p, at.s, rows, at.tiles, at.row_tiles);
}
// To the first tile of the next item; only where the list has one.
__device__ __forceinline__ void paged_next_item(const FaPagedParams& p, PagedCursor& at, int rows) {
  if (++at.rt < at.row_tiles) return;
  at.rt = 0;
  if (++at.h < p.c.Hkv) return;
  at.h = 0;
  do {
    if (++at.b >= p.c.B) return;
    paged_enter(p, at, rows);
  } while (at.row_tiles == 0);
}

template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kPagedThreads, 2) fa_paged_rows_kernel(const __grid_constant__ FaPagedParams p) {
  using Smem = FaPagedSmem<D, kRows>;
  constexpr bool kStacked = kRows == 8;              // A holds first parts over second parts
  constexpr bool kHalf = Pack2<T>::kFormat == 0;     // fp16: q is a sum of three
  constexpr float kLow = kStacked ? 16.f : 1.f;      // second parts are kept times this
  constexpr int kSteps = D / 32;                     // products along head_dim
  constexpr int kCols = D / 8;                       // accumulator tiles of O
  constexpr int kHalves = kRows / 8;                 // rows of a lane
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const KvView& kv = p.c;
  grid_launch_dependents();
  grid_wait();

  // ---- this block's run of the list
  long long mine = 0;
  for (int b = threadIdx.x; b < kv.B; b += kPagedThreads) {
    int tiles, row_tiles;
    mine += paged_list(p, kv_seq(kv, b), kRows, tiles, row_tiles);
    if (blockIdx.x == 0) {
      const uint32_t f = kv_seq_faults(kv, b);
      if (f != 0) kv_report(kv, f);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sm.sums[warp] = mine;
  if (threadIdx.x == 0) p.heads[blockIdx.x].last = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) total += sm.sums[w];
  if (total == 0) return;
  const int runs = paged_runs(total, gridDim.x), run = blockIdx.x;
  if (run >= runs) return;
  const long long begin = paged_begin(total, runs, run), end = paged_begin(total, runs, run + 1);
  long long before = 0;  // of the sequences in front of this round's
  for (int b0 = 0; b0 < kv.B && before <= begin; b0 += kPagedThreads) {
    const int b = b0 + threadIdx.x;
    int tiles, row_tiles;
    const long long own = b < kv.B ? paged_list(p, kv_seq(kv, b), kRows, tiles, row_tiles) : 0;
    long long upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    __syncthreads();
    if (lane == 31) sm.sums[warp] = upto;
    __syncthreads();
    long long at = before;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      if (w < warp) at += sm.sums[w];
      before += sm.sums[w];
    }
    if (at + upto > begin && at + upto - own <= begin) {
      sm.found = b;
      sm.found_at = at + upto - own;
    }
  }
  __syncthreads();

  PagedCursor seg;  // the segment's item and first tile
  seg.b = sm.found;
  paged_enter(p, seg, kRows);
  {
    const long long in = begin - sm.found_at;
    const long long item = in / seg.tiles;
    seg.j = static_cast<int>(in - item * seg.tiles);
    seg.h = static_cast<int>(item / seg.row_tiles);
    seg.rt = static_cast<int>(item - static_cast<long long>(seg.h) * seg.row_tiles);
  }

  // ---- loads: the warp's next tile, and the ids of the pages of the one after
  PagedCursor ld = seg;
  long long ld_left = end - begin - warp;  // tiles of the run from the next load on; the warp's are every fourth
  auto skip = [&](int tiles) {
    ld.j += tiles;
    while (ld.j >= ld.tiles && ld.b < kv.B) {
      ld.j -= ld.tiles;
      paged_next_item(p, ld, kRows);
    }
  };
  auto pages = [&](int& first, int& second) {  // of the tile's halves; -1: none of the cache's, or behind the sequence
    const int tok = ld.j * kPagedTile;
    first = tok < ld.s.len ? kv_page(kv, ld.b, tok >> kv.page_shift) : -1;
    second = tok + 16 < ld.s.len ? kv_page(kv, ld.b, (tok + 16) >> kv.page_shift) : -1;
  };
  int page0 = -1, page1 = -1;
  if (ld_left > 0) {
    skip(warp);
    pages(page0, page1);
  }
  uint32_t ld_stage = 0;
  auto load = [&]() {  // one tile, or nothing behind the run's end: a group of copies either way
    if (ld_left > 0) {
      const int tok = ld.j * kPagedTile;
      const uint32_t base = smem_u32(sm.ring[warp][ld_stage]);
      constexpr int kChunks = D / 16;          // of a row
      constexpr int kRowsAtOnce = 32 / kChunks;
      const int chunk = lane % kChunks;
#pragma unroll
      for (int i = 0; i < kPagedTile / kRowsAtOnce; ++i) {
        const int row = i * kRowsAtOnce + lane / kChunks;
        const int page = row < 16 ? page0 : page1;
        const bool real = page >= 0 && tok + row < ld.s.len;
        const int place = (tok + row) & ((1 << kv.page_shift) - 1);
        const int sw = D == 128 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
        const uint8_t* ks = real ? kv.k + page * kv.k_sp + ld.h * kv.k_sh + place * kv.k_ss + chunk * 16 : kv.k;
        const uint8_t* vs = real ? kv.v + page * kv.v_sp + ld.h * kv.v_sh + place * kv.v_ss + chunk * 16 : kv.v;
        cp_async16(base + row * D + sw * 16, ks, real);
        cp_async16(base + Smem::kTileBytes + row * D + sw * 16, vs, real);
      }
      if (lane < 4) {
        const int page = lane & 1 ? page1 : page0;
        const float* src = (lane & 2 ? kv.v_scale : kv.k_scale) + (page >= 0 ? static_cast<long long>(page) * kv.Hkv + ld.h : 0);
        cp_async4(smem_u32(&sm.scales[warp][ld_stage][lane]), src, page >= 0);
        if (page < 0 && tok + 16 * (lane & 1) < ld.s.len) kv_report(kv, HB_CACHE_BAD_PAGE);
      }
      if (++ld_stage == Smem::kStages) ld_stage = 0;
      ld_left -= kPagedWarps;
      if (ld_left > 0) {
        skip(kPagedWarps);
        pages(page0, page1);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < Smem::kStages - 1; ++i) load();

  // ---- segments
  uint32_t stage = 0;
  int turn = 0;  // tiles of the run in front of the segment, modulo the warps
  bool first = true;
  for (long long t = begin; t < end;) {
    const long long left = end - t;
    const int j0 = seg.j, j1 = left < seg.tiles - j0 ? j0 + static_cast<int>(left) : seg.tiles;
    const int rows = seg.s.n * p.group, row0 = seg.rt * kRows;

    // the lane's rows: their scaled queries in parts, and the keys they see
    uint32_t qa[kSteps][4], qb[kStacked ? (kHalf ? kSteps : 1) : kSteps][4], qc[(!kStacked && kHalf) ? kSteps : 1][4];
    float factor[kHalves];
    int limit[kHalves];
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      const int row = row0 + g + 8 * r;
      const bool live = row < rows;
      const int tok = live ? fast_div(row, p.by_group) : 0, head = live ? row - tok * p.group : 0;
      const T* src = static_cast<const T*>(p.q) + (seg.s.start + tok) * p.q_st + (seg.h * p.group + head) * p.q_sh;
      limit[r] = live ? (p.causal ? min(seg.s.len, seg.s.pos0() + tok + 1) : seg.s.len) : 0;
      float x[D / 64][16];
      float top = 0.f;
      bool finite = true;
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) {
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if (live) w = *reinterpret_cast<const uint4*>(src + 64 * hh + 16 * c + e);
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
      // 2^up takes the largest element into (224, 448]; a row that holds an infinity or NaN is NaN
      int up = 0;
      if (top > 0.f && top <= 3.402823466e38f) {
        const int bits = __float_as_int(top);
        up = 8 - ((bits >> 23) - 127) - ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
        up = min(max(up, -120), 120);
      }
      const float mul = __int_as_float((up + 127) << 23);
      const unsigned votes = __ballot_sync(0xffffffffu, finite);
      factor[r] = ((votes >> (lane & ~3)) & 15u) == 15u ? p.scale_log2 * __int_as_float((127 - up) << 23) : __int_as_float(0x7fc00000);
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = x[st >> 1][8 * (st & 1) + 4 * half + e] * mul;
          const uint32_t a = e4m3_part4(y);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= kLow;
          const uint32_t b = e4m3_part4(y);
          const uint32_t d = e4m3_last(y[0], y[1]) | (e4m3_last(y[2], y[3]) << 16);
          if constexpr (kStacked) {
            qa[st][2 * half] = a;
            qa[st][2 * half + 1] = b;
            if constexpr (kHalf) {
              qb[st][2 * half] = 0u;
              qb[st][2 * half + 1] = d;
            }
          } else {
            qa[st][2 * half + r] = a;
            qb[st][2 * half + r] = b;
            if constexpr (kHalf) qc[st][2 * half + r] = d;
          }
        }
      }
    }
    // keys that every live row sees: the first row's token sees least
    const int least = p.causal ? min(seg.s.len, seg.s.pos0() + fast_div(row0, p.by_group) + 1) : seg.s.len;

    float o[kCols][4];
#pragma unroll
    for (int i = 0; i < kCols; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[kHalves], l[kHalves], v_ref = 0.f;  // v_ref: O is in units of it / 256
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }

    for (int j = j0 + ((warp - turn) & (kPagedWarps - 1)); j < j1; j += kPagedWarps) {
      cp_async_wait<Smem::kStages - 2>();
      __syncwarp();  // every lane's copies are there, and every lane is done with the tile before: its stage is free
      load();
      const uint8_t* tile = sm.ring[warp][stage];
      const float ks[2] = {sm.scales[warp][stage][0], sm.scales[warp][stage][1]};
      const float vs[2] = {sm.scales[warp][stage][2], sm.scales[warp][stage][3]};

      // scores of the 32 keys: column n of group i is key 8 i + (n ^ 4 (n & 1))
      float x[4][2 * kHalves];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 8 * i + (g ^ ((g & 1) << 2));
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hh = 0; hh < D / 64; ++hh) {
          const int chunk = c + 4 * hh;
          const int sw = D == 128 ? chunk ^ (key & 7) : chunk ^ ((key >> 1) & 3);
          const uint4 k4 = *reinterpret_cast<const uint4*>(tile + key * D + sw * 16);
          const int st = 2 * hh;
          mma_e4m3(s, qa[st][0], qa[st][1], qa[st][2], qa[st][3], k4.x, k4.y);
          mma_e4m3(s, qa[st + 1][0], qa[st + 1][1], qa[st + 1][2], qa[st + 1][3], k4.z, k4.w);
          if constexpr (!kStacked || kHalf) {
            mma_e4m3(s, qb[st][0], qb[st][1], qb[st][2], qb[st][3], k4.x, k4.y);
            mma_e4m3(s, qb[st + 1][0], qb[st + 1][1], qb[st + 1][2], qb[st + 1][3], k4.z, k4.w);
          }
          if constexpr (!kStacked && kHalf) {
            mma_e4m3(s, qc[st][0], qc[st][1], qc[st][2], qc[st][3], k4.x, k4.y);
            mma_e4m3(s, qc[st + 1][0], qc[st + 1][1], qc[st + 1][2], qc[st + 1][3], k4.z, k4.w);
          }
        }
        if constexpr (kStacked) {
          x[i][0] = s[0] + s[2] * (1.f / kLow);
          x[i][1] = s[1] + s[3] * (1.f / kLow);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][e] = s[e];
        }
      }
      const bool masked = (j + 1) * kPagedTile > least || ks[0] == 0.f || ks[1] == 0.f;
      float pv[2] = {0.f, 0.f};  // 256 vscale / v_ref of the halves
      float shrink_o = 1.f;
      {
        const float top = fmaxf(vs[0], vs[1]);
        if (top > v_ref) {
          shrink_o = v_ref / top;  // powers of two (0 at first, where O is 0)
          v_ref = top;
        }
        if (v_ref > 0.f) {
          pv[0] = 256.f * (vs[0] / v_ref);
          pv[1] = 256.f * (vs[1] / v_ref);
        }
      }
      bool moved = shrink_o != 1.f;
      float alpha[kHalves];
#pragma unroll
      for (int r = 0; r < kHalves; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = factor[r] * ks[i >> 1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s = x[i][2 * r + e];
            s *= f;
            if (masked) {
              const int n = 2 * c + e, key = j * kPagedTile + 8 * i + (n ^ (e << 2));
              if (key >= limit[r] || ks[i >> 1] == 0.f) s = -INFINITY;
            }
            top = fmaxf(top, s);
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(m[r], top);
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        alpha[r] = fast_exp2(m[r] - m_safe);  // 0 while m is -inf, as O and l are
        moved = moved || (m_new != m[r]);
        m[r] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& s = x[i][2 * r + e];
            s = fast_exp2(s - m_safe);
            sum += s;
            s *= pv[i >> 1];
          }
        }
        l[r] = l[r] * alpha[r] + sum;
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float f0 = alpha[0] * shrink_o, f1 = (kStacked ? alpha[0] : alpha[kHalves - 1]) * shrink_o;
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
          o[i][0] *= f0;
          o[i][1] *= f0;
          o[i][2] *= f1;
          o[i][3] *= f1;
        }
      }
      // P in parts, as A: columns 4 c .. of the first 16 keys are columns 2 c, 2 c + 1 of score groups 0 and 1
      uint32_t pa[4], pb[4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {
          float y[4] = {x[2 * half][2 * r], x[2 * half][2 * r + 1], x[2 * half + 1][2 * r], x[2 * half + 1][2 * r + 1]};
          const uint32_t a = e4m3_part4(y);
          const uint32_t b = e4m3_last(y[0] * kLow, y[1] * kLow) | (e4m3_last(y[2] * kLow, y[3] * kLow) << 16);
          if constexpr (kStacked) {
            pa[2 * half] = a;
            pa[2 * half + 1] = b;
          } else {
            pa[2 * half + r] = a;
            pb[2 * half + r] = b;
          }
        }
      }
      // O += P V: the lane's value rows are keys 2 c, (2 c + 1) ^ 4, and those plus 8 of either half; its columns D / 8 from D / 8 g on
      constexpr int kWords = D / 32;  // of 4 columns
      uint32_t vw[2][4][kWords];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 2 * c + (i & 1);
          const int key = 16 * half + 8 * (i >> 1) + (n ^ ((i & 1) << 2));
          const uint8_t* row = tile + Smem::kTileBytes + key * D;
          if constexpr (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(row + ((g ^ (key & 7)) * 16));
            vw[half][i][0] = w.x;
            vw[half][i][1] = w.y;
            vw[half][i][2] = w.z;
            vw[half][i][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(row + (((g >> 1) ^ ((key >> 1) & 3)) * 16) + (g & 1) * 8);
            vw[half][i][0] = w.x;
            vw[half][i][1] = w.y;
          }
        }
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t b[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t t0 = __byte_perm(vw[half][0][w], vw[half][1][w], 0x5140), t1 = __byte_perm(vw[half][2][w], vw[half][3][w], 0x5140);
          const uint32_t t2 = __byte_perm(vw[half][0][w], vw[half][1][w], 0x7362), t3 = __byte_perm(vw[half][2][w], vw[half][3][w], 0x7362);
          b[half][0] = __byte_perm(t0, t1, 0x5410);
          b[half][1] = __byte_perm(t0, t1, 0x7632);
          b[half][2] = __byte_perm(t2, t3, 0x5410);
          b[half][3] = __byte_perm(t2, t3, 0x7632);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mma_e4m3(o[4 * w + e], pa[0], pa[1], pa[2], pa[3], b[0][e], b[1][e]);
          if constexpr (!kStacked) mma_e4m3(o[4 * w + e], pb[0], pb[1], pb[2], pb[3], b[0][e], b[1][e]);
        }
      }
      if (++stage == Smem::kStages) stage = 0;
    }

    // ---- the warps' results meet
    const float unit = v_ref * (1.f / 256.f);
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c == 0) {
        sm.ml[warp][0][g + 8 * r] = m[r];
        sm.ml[warp][1][g + 8 * r] = l[r];
      }
    }
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {  // columns n = 2 c + e2: D / 8 n + 4 w + 0 .. 3
        const int col = (D / 8) * (2 * c + e2) + 4 * w;
        if constexpr (kStacked) {
          float4 y;
          y.x = (o[4 * w][e2] + o[4 * w][2 + e2] * (1.f / kLow)) * unit;
          y.y = (o[4 * w + 1][e2] + o[4 * w + 1][2 + e2] * (1.f / kLow)) * unit;
          y.z = (o[4 * w + 2][e2] + o[4 * w + 2][2 + e2] * (1.f / kLow)) * unit;
          y.w = (o[4 * w + 3][e2] + o[4 * w + 3][2 + e2] * (1.f / kLow)) * unit;
          *reinterpret_cast<float4*>(&sm.o[warp][g][col]) = y;
        } else {
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *reinterpret_cast<float4*>(&sm.o[warp][g + 8 * r][col]) =
                make_float4(o[4 * w][2 * r + e2] * unit, o[4 * w + 1][2 * r + e2] * unit, o[4 * w + 2][2 * r + e2] * unit,
                            o[4 * w + 3][2 * r + e2] * unit);
        }
      }
    }
    __syncthreads();
    const bool whole = j0 == 0 && j1 == seg.tiles;
    const int slot = 2 * run + (first ? 0 : 1);
    for (int i = threadIdx.x; i < kRows * (D / 8); i += kPagedThreads) {
      const int r = i / (D / 8), col = i % (D / 8) * 8, row = row0 + r;
      if (row >= rows) continue;
      float top = sm.ml[0][0][r];
#pragma unroll
      for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, sm.ml[w][0][r]);
      const float safe = top == -INFINITY ? 0.f : top;
      float sum = 0.f, y[8] = {};
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const float wt = fast_exp2(sm.ml[w][0][r] - safe);
        sum += wt * sm.ml[w][1][r];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 z = *reinterpret_cast<const float4*>(&sm.o[w][r][col + e]);
          y[e] += wt * z.x;
          y[e + 1] += wt * z.y;
          y[e + 2] += wt * z.z;
          y[e + 3] += wt * z.w;
        }
      }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;  // a row without keys is 0, one with a NaN is NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= inv;
      const float lse2 = sum != 0.f ? safe + fast_log2(sum) : -INFINITY;
      if (whole) {
        const int tok = fast_div(row, p.by_group), head = seg.h * p.group + row - tok * p.group;
        T* dst = static_cast<T*>(p.o) + (seg.s.start + tok) * p.o_st + head * p.o_sh + col;
        uint4 w4;
        w4.x = Pack2<T>::pack(y[0], y[1]);
        w4.y = Pack2<T>::pack(y[2], y[3]);
        w4.z = Pack2<T>::pack(y[4], y[5]);
        w4.w = Pack2<T>::pack(y[6], y[7]);
        *reinterpret_cast<uint4*>(dst) = w4;
        if (col == 0 && p.lse != nullptr) p.lse[static_cast<long long>(seg.s.start + tok) * p.Hq + head] = lse2 * 0.6931471805599453f;
      } else {
        float* dst = p.part_o + (static_cast<long long>(slot) * kRows + r) * D + col;
        *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
        if (col == 0) p.part_lse[static_cast<long long>(slot) * kRows + r] = lse2;
      }
    }
    if (threadIdx.x == 0 && j0 == 0 && !whole) {
      PagedHead& hd = p.heads[run];
      hd.b = seg.b;
      hd.h = seg.h;
      hd.rt = seg.rt;
      hd.slot = slot;
      hd.last = paged_run_of(total, runs, t + seg.tiles - 1);
    }
    __syncthreads();
    turn = (turn + (j1 - j0)) & (kPagedWarps - 1);
    t += j1 - j0;
    first = false;
    seg.j = 0;
    if (t < end) paged_next_item(p, seg, kRows);
  }
  cp_async_wait<0>();
}

// Merges the parts of an item: one block per (run that starts an item in parts, row); its warps deal the parts out, a lane has
// D / 32 columns; weights 2^(lse - max).
constexpr int kPagedCombineWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kPagedCombineWarps) fa_paged_combine_kernel(const __grid_constant__ FaPagedParams p, int kRows) {
  grid_launch_dependents();
  grid_wait();
  const int run = blockIdx.x / kRows, r = blockIdx.x - run * kRows;
  const PagedHead hd = p.heads[run];
  if (hd.last < 0) return;
  const KvSeq s = kv_seq(p.c, hd.b);
  const int row = hd.rt * kRows + r;
  if (row >= s.n * p.group) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  auto slot_of = [&](int w) -> long long { return w == run ? hd.slot : 2 * w; };

  float top = -INFINITY;
  for (int w = run + lane; w <= hd.last; w += 32) top = fmaxf(top, p.part_lse[slot_of(w) * kRows + r]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;

  constexpr int kCols = D / 32;
  float acc[kCols] = {}, sum = 0.f;
#pragma unroll 4
  for (int w = run + warp; w <= hd.last; w += warps) {
    const long long at = slot_of(w) * kRows + r;
    const float wt = fast_exp2(p.part_lse[at] - top);
    const float* src = p.part_o + at * D + lane * kCols;
    sum += wt;
    if constexpr (kCols == 4) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      acc[0] += wt * x.x;
      acc[1] += wt * x.y;
      acc[2] += wt * x.z;
      acc[3] += wt * x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(src);
      acc[0] += wt * x.x;
      acc[1] += wt * x.y;
    }
  }
  __shared__ float s_acc[kPagedCombineWarps][D], s_sum[kPagedCombineWarps];
#pragma unroll
  for (int e = 0; e < kCols; ++e) s_acc[warp][lane * kCols + e] = acc[e];
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
  sum = 0.f;
  for (int k = 0; k < warps; ++k) sum += s_sum[k];
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  uint32_t packed[kCols / 2];
#pragma unroll
  for (int e = 0; e < kCols; e += 2) {
    float a = 0.f, b = 0.f;
    for (int k = 0; k < warps; ++k) {
      a += s_acc[k][lane * kCols + e];
      b += s_acc[k][lane * kCols + e + 1];
    }
    packed[e / 2] = Pack2<T>::pack(a * inv, b * inv);
  }
  const int tok = fast_div(row, p.by_group), head = hd.h * p.group + row - tok * p.group;
  T* dst = static_cast<T*>(p.o) + (s.start + tok) * p.o_st + head * p.o_sh + lane * kCols;
  if constexpr (kCols == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  else *reinterpret_cast<uint32_t*>(dst) = packed[0];
  if (lane == 0 && p.lse != nullptr)
    p.lse[static_cast<long long>(s.start + tok) * p.Hq + head] = (sum != 0.f ? top + fast_log2(sum) : -INFINITY) * 0.6931471805599453f;
}

}  // namespace hb
