// Attention of many query rows (prompts, chunks of them) over the paged 8-bit cache (hb_fa_paged), sm_100a.
//
// Bound by the tensor cores and the exponentials, as fa_fwd: 256 query rows of one (sequence, KV head) a block, row = token * group +
// head, against key tiles of 128, S and O in TMEM, P over S.  What differs is what feeds it:
//   - four producer warps fetch the codes of a tile's pages (whatever their order), convert them to fp16 and store them as the
//     operands that tcgen05.mma reads (128-byte swizzle; keys K-major, values MN-major), each tile once for 256 rows.  Two
//     e4m3 products of a query's and a weight's parts would need no conversion, and twice the products and a split of every weight;
//   - the scales of a tile's pages are taken relative to the tile's largest, powers of two that fp16 holds beside the code; where all
//     are alike, nearly always, nothing is multiplied.  The largest goes into the factor of the scores and into the weights P'.  Where
//     scales of a tile are more than 2^8 apart its codes stay as they are, and the softmax has the scales of every 16 keys;
//   - queries are scaled into fp16 by a power of two for each row, by the thread that owns the row.
// An item's key tiles are dealt out to several blocks where items are few, or do not fill the SMs evenly (paged_splits); their fp32 partial
// results meet in fa_paged_tiles_combine_kernel.
// A row's maximum is that of score + log2 value scale, adopted when it grew by more than 2^7 (fa_paged_sm100.cuh).  O is rescaled by the row's
// own thread, as in fa_split.
//
// us in a captured graph: B2 Hq32 Hkv8 D128, 2048 queries behind 6144 507 (0.93 PFLOP/s; tensor pipe and MUFU 48 % each); B4 Hq16
// Hkv16 D64, prompts of 1024 33.9; B16 Hq28 Hkv4 D128, 1 to 400 queries behind 750 to 1500 105.3.  The short ones pay for starts and ends of blocks.
#pragma once

#include "fa_fwd_sm100.cuh"
#include "fa_paged_sm100.cuh"

namespace hb {

constexpr int kPagedTilesThreads = 512;  // 8 softmax warps, the MMA warp (and three idle ones), 4 producers
constexpr int kPagedBlockRows = 2 * kTileM;
enum FaPagedRole : uint32_t { kRolePagedSoftmax = 10, kRolePagedMma = 11, kRolePagedProducer = 12, kRolePagedDrain = 13 };

struct FaPagedTilesParams {
  KvView c;
  const void* q;
  void* o;
  float* lse;
  long long q_st, q_sh, o_st, o_sh;
  int Hq, group, causal;
  int row_limit;  // sequences with no more query rows a KV head are the rows kernel's
  FastDiv by_group, by_hkv, by_b;
  float scale_log2;
  uint32_t* status;
  int splits;       // blocks of the grid for an item: each has a part of its key tiles
  float* part_o;    // splits > 1: [grid][256][D], O / l of the part
  float* part_lse;  // [grid][256], base 2; -inf: no keys
  struct PagedParts* parts;  // [grid / splits]
};

struct alignas(16) PagedParts {  // of an item
  int count;                // 0: no item, 1: its block has stored the rows
  int h, row0, rows, start, pad[3];
};

template <int D>
struct FaPagedTilesSmem {
  static constexpr int kTileBytes = kTileN * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 10;
  alignas(1024) uint8_t q[2][kTileBytes];
  alignas(1024) uint8_t kv[kStages][kTileBytes];
  static constexpr int kMeta = 8;
  // K(j + kMeta) takes the ring's place of tile 2 (j + kMeta) - kStages of K(0) V(0) K(1) V(1) ..: where that is V(j) or later, P(j) was
  // there, and so meta(j) read
  static_assert(2 * kMeta - kStages >= 1, "a tile's scales are overwritten only when its softmax is done");
  float4 meta[kMeta];  // of key tile j at j % kMeta: largest key scale, largest value scale, bits of groups of 16 keys that are not there, 1: ...
  float2 group[kMeta][kTileN / 16];  // ... the codes are as they are, and these the scales of keys and values
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t meta_full[kMeta];
  uint64_t drain;
  long long sums[kPagedTilesThreads / 32];
  long long found_at;
  int found, descends;
  uint32_t tmem_base;
  uint32_t abort_flag;
};

struct PagedItem {
  KvSeq s;
  int b, h, row0, rows;  // rows of the sequence in this KV head
  int j0, j1;            // key tiles of the block
  int n[2];              // of them, row tile i has [j0, n[i])
  bool whole;            // all of the item's
};

__device__ __forceinline__ int paged_blocks_of(const FaPagedTilesParams& p, const KvSeq& s) {
  const long long rows = static_cast<long long>(s.n) * p.group;
  return rows > p.row_limit ? static_cast<int>((rows + kPagedBlockRows - 1) / kPagedBlockRows) : 0;
}

// Rows of q and o are read and written by D / 8 lanes each, whole rows an access, through the places of the queries in shared memory; by
// their owners a block's start took 8300 cycles for the queries.
template <int D>
struct PagedRows {
  static constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
  uint8_t* base;
  int warp_row, sub, piece;
  __device__ __forceinline__ PagedRows(FaPagedTilesSmem<D>& s, int i)
      : base(s.q[i]), warp_row(threadIdx.x & (kTileM - 1) & ~31), sub((threadIdx.x & 31) / kLanes), piece(threadIdx.x % kLanes) {}
  // chunk e of row x, where the matrix instruction reads the queries
  __device__ __forceinline__ uint4* at(int x, int e) const {
    return reinterpret_cast<uint4*>(base + (e >> 3) * (kTileM * 128) + x * 128 + ((e & 7) ^ (x & 7)) * 16);
  }
  __device__ __forceinline__ uint4* mine(int k) const { return at(warp_row + k * kAtOnce + sub, piece); }  // k < kLanes
  // its place in global memory, from the owner's place of the row; kNone: not a row of the sequence (strides may be negative)
  static constexpr long long kNone = -0x7fffffffffffffffll - 1;
  __device__ __forceinline__ long long place(int k, long long own) const {
    const long long row = __shfl_sync(0xffffffffu, own, k * kAtOnce + sub);
    return row == kNone ? kNone : row + 8 * piece;
  }
};

// The queries as they are; the softmax warps wait for them and scale them in place.
template <typename T, int D>
__device__ __forceinline__ void paged_copy_queries(const FaPagedTilesParams& p, FaPagedTilesSmem<D>& s, const PagedItem& it, int i) {
  if ((i == 0 ? it.n[0] : it.n[1]) <= it.j0) return;
  const PagedRows<D> rows(s, i);
  const int row = it.row0 + kTileM * i + static_cast<int>(threadIdx.x & (kTileM - 1));
  const int tok = fast_div(row, p.by_group);
  const long long own = row < it.rows ? (it.s.start + tok) * p.q_st + (it.h * p.group + row - tok * p.group) * p.q_sh : PagedRows<D>::kNone;
#pragma unroll 4
  for (int k = 0; k < PagedRows<D>::kLanes; ++k) {
    const long long at = rows.place(k, own);
    const bool real = at != PagedRows<D>::kNone;
    cp_async16(smem_u32(rows.mine(k)), static_cast<const T*>(p.q) + (real ? at : 0ll), real);
  }
}

// A value scale relative to `base`, both by their bits: the difference of the exponents in place.  0 where the scale is: values are 0 then.
__device__ __forceinline__ int paged_relative(float scale, int base) {
  return scale != 0.f ? min(max(__float_as_int(scale) - base, -(126 << 23)), 126 << 23) : 0;
}
__device__ __forceinline__ float paged_log(int to) { return static_cast<float>(to >> 23); }
__device__ __forceinline__ float paged_inverse(int to) { return __int_as_float((127 << 23) - to); }

// A tile whose scales are far apart: scores with the scales of their groups.  In short loops that read the scores again, 32 at a time, and in one
// piece beside the usual path: with a branch in front of the maximum and one in front of the weights, that path took ragged batches
// from 106 to 113 us without a single such tile.
// Scores of 32 keys, of which half h has group 2 q + h.
__device__ __forceinline__ void paged_group_scores(uint32_t tS, const float2* group, float factor, int lim, int q, uint32_t (&x)[32], float2 (&scale)[2],
                                                   float (&f)[2]) {
  tmem_ld32(tS + q * 32, x);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    scale[h] = group[2 * q + h];
    f[h] = factor * scale[h].x;
    f[h] = f[h] == 0.f ? 1.17549435e-38f : f[h];
  }
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < 32; ++c) x[c] = q * 32 + c <= lim && scale[c >> 4].x != 0.f ? x[c] : 0xff800000u;
}
// The row's new maximum and sum, and what it falls by; P' goes to its place, which is that of scores that are read already: 16 columns for 32.
__device__ __forceinline__ float3 paged_group_softmax(uint32_t tS, const float2* group, float factor, int lim, int base, bool live, float m, float l) {
  float top = -INFINITY;
#pragma unroll 1
  for (int q = 0; q < kTileN / 32; ++q) {
    uint32_t x[32];
    float2 scale[2];
    float f[2];
    paged_group_scores(tS, group, factor, lim, q, x, scale, f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = __uint_as_float(x[16 * h]);
#pragma unroll
      for (int c = 1; c < 16; ++c) mx = fmaxf(mx, __uint_as_float(x[16 * h + c]));
      top = fmaxf(top, fmaf(mx, f[h], paged_log(paged_relative(scale[h].y, base))));
    }
  }
  const bool adopt = live && top > m + kPagedGrowth;
  const float alpha = adopt ? fast_exp2(m - top) : 1.f;
  m = adopt ? top : m;
  l *= alpha;
  const float off = kPagedBits - (m == -INFINITY ? 0.f : m);
#pragma unroll 1
  for (int q = 0; q < kTileN / 32; ++q) {
    uint32_t x[32], pk[16];
    float2 scale[2];
    float f[2];
    paged_group_scores(tS, group, factor, lim, q, x, scale, f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int to = paged_relative(scale[h].y, base);
      const float off_h = off + paged_log(to);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 16; c += 2) {
        const float a = fast_exp2(fmaf(__uint_as_float(x[16 * h + c]), f[h], off_h));
        const float b = fast_exp2(fmaf(__uint_as_float(x[16 * h + c + 1]), f[h], off_h));
        sum += a + b;
        pk[8 * h + c / 2] = scale[h].y != 0.f ? Pack2<__half>::pack(a, b) : 0u;
      }
      l = fmaf(sum, paged_inverse(to), l);
    }
    tmem_st16(tS + q * 16, pk);
  }
  return make_float3(m, l, alpha);
}

template <typename T, int D>
__device__ __forceinline__ void paged_softmax_role(const FaPagedTilesParams& p, FaPagedTilesSmem<D>& s, const AbortCtx& ctx, uint32_t tmem,
                                                   const PagedItem& it, int i) {
  using Smem = FaPagedTilesSmem<D>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = threadIdx.x & (kTileM - 1);
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + lane_off + static_cast<uint32_t>(i * kTileN), tO = tmem + lane_off + 256u + static_cast<uint32_t>(i * 128);
  const int n = i == 0 ? it.n[0] : it.n[1];
  const long long part_row = static_cast<long long>(blockIdx.x) * kPagedBlockRows + kTileM * i + r;
  if (n <= it.j0) {
    if (!it.whole) p.part_lse[part_row] = -INFINITY;
    return;
  }
  const int first = it.row0 + kTileM * i, row = first + r;
  const bool live = row < it.rows;
  const int tok = live ? fast_div(row, p.by_group) : 0, head = it.h * p.group + (live ? row - tok * p.group : 0);
  const int limit = !live ? 0 : p.causal ? min(it.s.len, it.s.pos0() + tok + 1) : it.s.len;
  const int least = p.causal ? min(it.s.len, it.s.pos0() + fast_div(first, p.by_group) + 1) : it.s.len;

  const PagedRows<D> rows(s, i);
  float factor;
  {  // the queries in fp16: 2^up takes a row's largest element into [2^14, 2^15)
    cp_async_wait<0>();
    __syncwarp();
    uint32_t tops = 0u;  // without their signs, 16-bit numbers are in the order of their bits, infinities and NaN above all others
#pragma unroll
    for (int e = 0; e < D / 8; ++e) {
      const uint4 w = *rows.at(r, e);
      tops = __vimax3_u16x2(tops, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
      tops = __vimax3_u16x2(tops, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu);
    }
    float top, none;
    Pack2<T>::unpack(max(tops & 0xffffu, tops >> 16), top, none);
    const bool finite = top <= 3.402823466e38f;
    int up = 0;
    if (top > 0.f && finite) up = min(14 - ((__float_as_int(top) >> 23) - 127), 120);
    // a row that holds an infinity or NaN is NaN: its scores are, those of keys that it sees
    const float mul = finite ? __int_as_float((up + 127) << 23) : __int_as_float(0x7fc00000);
    factor = p.scale_log2 * __int_as_float((127 - up) << 23);
#pragma unroll
    for (int e = 0; e < D / 8; ++e) {
      const uint4 w = *rows.at(r, e);
      uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        Pack2<T>::unpack(u[k], a, b);
        u[k] = Pack2<__half>::pack(a * mul, b * mul);
      }
      *rows.at(r, e) = make_uint4(u[0], u[1], u[2], u[3]);
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.q_full[i]);
  }

  // relative to `base`, the first tile's largest value scale; l in 2^(m - kPagedBits), O in that times base
  float m = -INFINITY, l = 0.f;
  int base = 0;  // bits; 0: no tile yet
  for (int j = it.j0; j < n; ++j) {
    const int at = j - it.j0;
    if (!mbar_wait_warp(&s.s_full[i], at & 1, ctx, kRolePagedSoftmax)) return;
    tc_fence_after();
    uint32_t v[kTileN];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, &v[c * 32]);
    if (!mbar_wait_warp(&s.meta_full[at % Smem::kMeta], (at / Smem::kMeta) & 1, ctx, kRolePagedSoftmax)) return;
    const float4 meta = s.meta[at % Smem::kMeta];
    const uint32_t gone = __float_as_uint(meta.z);
    tmem_wait_ld();

    if (base == 0) base = __float_as_int(meta.y);
    const int col0 = j * kTileN, lim = limit - 1 - col0;
    float alpha;
    if (meta.w != 0.f) {
      const float3 r = paged_group_softmax(tS, s.group[at % Smem::kMeta], factor, lim, base, live, m, l);
      m = r.x;
      l = r.y;
      alpha = r.z;
    } else {
      if (col0 + kTileN > least || gone != 0u) {
#pragma unroll
        for (int c = 0; c < kTileN; ++c) v[c] = (c <= lim && !((gone >> (c >> 4)) & 1u)) ? v[c] : 0xff800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) mx[c] = __uint_as_float(v[c]);
#pragma unroll
      for (int c = 4; c < kTileN; c += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c + 4 < kTileN) mx[e] = max3(mx[e], __uint_as_float(v[c + e]), __uint_as_float(v[c + 4 + e]));
          else mx[e] = fmaxf(mx[e], __uint_as_float(v[c + e]));
        }
      }
      float f = factor * meta.x;
      f = f == 0.f ? 1.17549435e-38f : f;  // -inf has to stay it
      const int to = paged_relative(meta.y, base);
      const float v_log = paged_log(to);
      const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), f, v_log);
      const bool adopt = live && top > m + kPagedGrowth;  // padding rows never ask for a rescale
      alpha = adopt ? fast_exp2(m - top) : 1.f;
      m = adopt ? top : m;
      const float off = v_log + kPagedBits - (m == -INFINITY ? 0.f : m);

      const uint64_t f2 = pack_f32x2(f, f), off2 = pack_f32x2(off, off);
      uint64_t sa = pack_f32x2(0.f, 0.f), sb = sa;
#pragma unroll
      for (int q = 0; q < kTileN / 32; ++q) {
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const int c = q * 32 + k;
          const uint64_t x0 = fma_f32x2(pack_f32x2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), f2, off2);
          const uint64_t x1 = fma_f32x2(pack_f32x2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), f2, off2);
          float a0, a1, b0, b1;
          unpack_f32x2(x0, a0, a1);
          unpack_f32x2(x1, b0, b1);
          a0 = fast_exp2(a0);
          a1 = fast_exp2(a1);
          b0 = fast_exp2(b0);
          b1 = fast_exp2(b1);
          sa = add_f32x2(sa, pack_f32x2(a0, a1));
          sb = add_f32x2(sb, pack_f32x2(b0, b1));
          pk[k / 2] = Pack2<__half>::pack(a0, a1);
          pk[k / 2 + 1] = Pack2<__half>::pack(b0, b1);
        }
        tmem_st16(tS + q * 16, pk);
      }
      float sum0, sum1, sum2, sum3;
      unpack_f32x2(sa, sum0, sum1);
      unpack_f32x2(sb, sum2, sum3);
      l = fmaf((sum0 + sum1) + (sum2 + sum3), paged_inverse(to), l * alpha);
    }
    // S(j) was committed behind P V(j - 1), so that product is complete, and P V(j) is only issued after this warp's arrival
    if (at > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
        tmem_st32(tO + c * 32, o);
      }
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.p_full[i]);
  }

  if (!mbar_wait_warp(&s.o_full[i], 0, ctx, kRolePagedSoftmax)) return;
  tc_fence_after();
  const float inv = l != 0.f ? __int_as_float(base) / l : 0.f;  // a row without keys is 0, one with a NaN is NaN
  const float lse2 = l != 0.f ? (m == -INFINITY ? 0.f : m) + (fast_log2(l) - kPagedBits) : -INFINITY;
  float* part = p.part_o + (part_row - (r & 3)) * D;
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    __syncwarp();
    tmem_ld32(tO + c * 32, o);
    tmem_wait_ld();
    if (it.whole) {
      uint4 w[4];
      pack_row32<T>(o, inv, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) *rows.at(r, 4 * c + k) = w[k];  // the queries' products are complete
    } else {
      store_rows32_f32(part + c * 32, D, 4, o, inv);
    }
  }
  if (it.whole) {
    __syncwarp();
    const long long own = live ? (it.s.start + tok) * p.o_st + head * p.o_sh : PagedRows<D>::kNone;
#pragma unroll 4
    for (int k = 0; k < PagedRows<D>::kLanes; ++k) {
      const long long at = rows.place(k, own);
      if (at != PagedRows<D>::kNone) *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at) = *rows.mine(k);
    }
  }
  if (!it.whole) p.part_lse[part_row] = lse2;
  else if (live && p.lse != nullptr) p.lse[static_cast<long long>(it.s.start + tok) * p.Hq + head] = lse2 * 0.6931471805599453f;
}

template <int D>
__device__ __forceinline__ void paged_mma_role(FaPagedTilesSmem<D>& s, const AbortCtx& ctx, uint32_t tmem, const PagedItem& it) {
  using Smem = FaPagedTilesSmem<D>;
  constexpr uint32_t kFmt = Pack2<__half>::kFormat;
  constexpr uint32_t idesc_qk = make_idesc(kFmt, kTileM, kTileN, 0, 0);
  constexpr uint32_t idesc_pv = make_idesc(kFmt, kTileM, D, 0, 1);
  constexpr uint32_t kSub = kTileM * 128u >> 4;                   // next 64 columns of head_dim
  constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // see fa_mma_role
  constexpr uint32_t kLboK = (16u >> 4) << 16, kLboV = kSub << 16;
  constexpr uint32_t kTile16 = Smem::kTileBytes >> 4;
  auto desc = [](uint32_t lo) -> uint64_t { return (static_cast<uint64_t>(kDescHi) << 32) | lo; };
  const uint32_t q_lo = (smem_u32(s.q[0]) >> 4) | kLboK, kv_lo = smem_u32(s.kv[0]) >> 4;
  const bool leader = elect_one();
  auto commit = [&](uint64_t* bar) {
    if (leader) umma_commit(bar);
  };
  auto issue_qk = [&](int i, uint32_t slot) {
    const uint32_t qa = q_lo + static_cast<uint32_t>(i) * kTile16, ka = (kv_lo + slot * kTile16) | kLboK;
    if (leader) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = static_cast<uint32_t>(kk >> 2) * kSub + static_cast<uint32_t>(kk & 3) * 2u;
        umma_ss_f16(tmem + static_cast<uint32_t>(i * kTileN), desc(qa + off), desc(ka + off), idesc_qk, kk > 0 ? 1u : 0u);
      }
    }
  };
  auto issue_pv = [&](int i, uint32_t slot, uint32_t accumulate) {
    const uint32_t va = (kv_lo + slot * kTile16) | kLboV, tS = tmem + static_cast<uint32_t>(i * kTileN);
    if (leader) {
#pragma unroll
      for (int kk = 0; kk < kTileN / 16; ++kk)
        umma_ts_f16(tmem + 256u + static_cast<uint32_t>(i * 128), tS + static_cast<uint32_t>(kk * 8), desc(va + static_cast<uint32_t>(kk) * (16u * 128u >> 4)),
                    idesc_pv, kk > 0 ? 1u : accumulate);
    }
  };
  uint32_t slot = 0, phase = 0;
  auto advance = [&]() {
    if (++slot == Smem::kStages) {
      slot = 0;
      phase ^= 1;
    }
  };
  const int j0 = it.j0, nmax = it.j1;
  uint32_t slot_k = slot;
  if (!mbar_wait_warp(&s.kv_full[slot], phase, ctx, kRolePagedMma)) return;
  advance();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if ((i == 0 ? it.n[0] : it.n[1]) <= j0) continue;
    if (!mbar_wait_warp(&s.q_full[i], 0, ctx, kRolePagedMma)) return;
    tc_fence_after();
    issue_qk(i, slot_k);
    commit(&s.s_full[i]);
  }
  commit(&s.kv_empty[slot_k]);
  for (int j = j0; j < nmax; ++j) {
    const uint32_t slot_v = slot;
    if (!mbar_wait_warp(&s.kv_full[slot], phase, ctx, kRolePagedMma)) return;
    advance();
    const bool has_next = j + 1 < nmax;
    bool k_ready = false;
    slot_k = slot;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const int ni = i == 0 ? it.n[0] : it.n[1];
      if (j < ni) {
        if (!mbar_wait_warp(&s.p_full[i], (j - j0) & 1, ctx, kRolePagedMma)) return;
        tc_fence_after();
        issue_pv(i, slot_v, j > j0 ? 1u : 0u);
        if (j == ni - 1) commit(&s.o_full[i]);
      }
      if (j + 1 < ni) {
        if (!k_ready) {
          if (!mbar_wait_warp(&s.kv_full[slot], phase, ctx, kRolePagedMma)) return;
          tc_fence_after();
          k_ready = true;
        }
        issue_qk(i, slot_k);
        commit(&s.s_full[i]);
      }
    }
    commit(&s.kv_empty[slot_v]);
    if (has_next) {
      commit(&s.kv_empty[slot_k]);
      advance();
    }
  }
}

// Producer warp pw has rows 32 pw .. + 31 of every tile.  A quarter of a warp reads 64 bytes of two rows next to each other: their
// fp16 chunks then lie in all eight places of a 128-byte line.
template <int D>
__device__ __forceinline__ void paged_producer_role(const FaPagedTilesParams& p, FaPagedTilesSmem<D>& s, const AbortCtx& ctx,
                                                    const PagedItem& it, int pw) {
  using Smem = FaPagedTilesSmem<D>;
  constexpr int kRowsAtOnce = 512 / D, kCopies = 32 / kRowsAtOnce;
  const KvView& kv = p.c;
  const int lane = threadIdx.x & 31, quarter = lane >> 3, l8 = lane & 7;
  const int rr = D == 128 ? 2 * (quarter >> 1) + (l8 >> 2) : 2 * quarter + (l8 >> 2);
  const int ch = D == 128 ? 4 * (quarter & 1) + (l8 & 3) : (l8 & 3);  // 16 codes
  uint32_t dst[2][2];  // of the lane's two fp16 chunks; rows eight apart (one or two copies) have the same swizzle
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = 32 * pw + (k * kRowsAtOnce) % 8 + rr;
#pragma unroll
    for (int x = 0; x < 2; ++x) dst[k][x] = (ch >> 2) * (kTileN * 128) + row * 128 + ((2 * (ch & 3) + x) ^ (row & 7)) * 16;
  }
  const int nmax = it.j1, len = it.s.len;

  // of key tile j, in lane g < 8: page and scales of keys 16 g .. + 15 (-1 and 0: none of the cache's, or behind the sequence)
  auto page_of = [&](int j) -> int {
    const int tok = j * kTileN + 16 * l8;
    return j < nmax && tok < len ? kv_page(kv, it.b, tok >> kv.page_shift) : -1;
  };
  auto scale_of = [&](const float* scales, int page) -> float {
    return page >= 0 ? scales[static_cast<long long>(page) * kv.Hkv + it.h] : 0.f;
  };
  auto fetch = [&](const uint8_t* base, unsigned sp, unsigned ss, int j, int page, uint4 (&w)[kCopies]) {
    const int tok = j * kTileN + 32 * pw, at = tok & ((1 << kv.page_shift) - 1);
    const int page0 = __shfl_sync(0xffffffffu, page, 2 * pw), page1 = __shfl_sync(0xffffffffu, page, 2 * pw + 1);
    const uint8_t* p0 = base + kv_offset(page0, sp) + kv_offset(at + rr, ss) + ch * 16;
    const uint8_t* p1 = base + kv_offset(page1, sp) + kv_offset((kv.page_shift == 4 ? 0 : at + 16) + rr, ss) + ch * 16;
    const long long step = kv_offset(kRowsAtOnce, ss);
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      const int half = k / (kCopies / 2), k2 = k % (kCopies / 2);
      const bool real = (half == 0 ? page0 : page1) >= 0 && tok + k * kRowsAtOnce + rr < len;
      w[k] = real ? *reinterpret_cast<const uint4*>((half == 0 ? p0 : p1) + k2 * step) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto store = [&](uint32_t slot, const uint4 (&w)[kCopies], bool alike, __half2 r0, __half2 r1) {
    const uint32_t tile = smem_u32(s.kv[slot]);
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      uint32_t h[8];
#pragma unroll
      for (int x = 0; x < 4; ++x) codes_f16(u[x], h[2 * x], h[2 * x + 1]);
      if (!alike) {
        const __half2 r = k < kCopies / 2 ? r0 : r1;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h[x]), r);
          h[x] = *reinterpret_cast<const uint32_t*>(&y);
        }
      }
      constexpr int kSame = 8 / kRowsAtOnce;  // copies until the swizzle repeats: 2 (D 128), 1 (D 64)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + dst[k % kSame][x] + (k / kSame) * 8 * 128), "r"(h[4 * x]),
                     "r"(h[4 * x + 1]), "r"(h[4 * x + 2]), "r"(h[4 * x + 3])
                     : "memory");
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.kv_full[slot]);
  };

  const uint8_t* k_base = kv.k + kv_offset(it.h, kv.k_sh);
  const uint8_t* v_base = kv.v + kv_offset(it.h, kv.v_sh);
  uint32_t slot = 0, phase = 1;  // "empty" barriers start out free
  auto advance = [&]() {
    if (++slot == Smem::kStages) {
      slot = 0;
      phase ^= 1;
    }
  };
  int page = page_of(it.j0);
  float ks = scale_of(kv.k_scale, page), vs = scale_of(kv.v_scale, page);
  uint4 wk[kCopies], wv[kCopies];
  fetch(k_base, kv.k_sp, kv.k_ss, it.j0, page, wk);
  for (int j = it.j0; j < nmax; ++j) {
    const int at = (j - it.j0) % Smem::kMeta;
    const int next = page_of(j + 1);
    fetch(v_base, kv.v_sp, kv.v_ss, j, page, wv);
    // the tile's largest scales, and this warp's two halves relative to them
    if (ks == 0.f) vs = 0.f;
    float k_ref = ks, v_ref = vs;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      k_ref = fmaxf(k_ref, __shfl_xor_sync(0xffffffffu, k_ref, o));
      v_ref = fmaxf(v_ref, __shfl_xor_sync(0xffffffffu, v_ref, o));
    }
    const float k_inv = k_ref > 0.f ? 1.f / k_ref : 0.f, v_inv = v_ref > 0.f ? 1.f / v_ref : 0.f;
    const bool inside = j * kTileN + 16 * l8 < len;
    const uint32_t gone = __ballot_sync(0xffffffffu, inside && ks == 0.f) & 0xffu;
    // 2^8 apart: fp16 holds the products, and takes P' no further down than that where a row does not see the largest
    bool k_alike = __all_sync(0xffffffffu, ks == 0.f || ks == k_ref);
    bool v_alike = __all_sync(0xffffffffu, (vs == v_ref && vs != 0.f) || page < 0);
    bool apart = false;
    if (!(k_alike && v_alike)) {  // asked only here: D128 chunks with pages of 16 133.6 us, with the question in front of every tile 136.9
      apart = __any_sync(0xffffffffu, (ks != 0.f && ks * 256.f < k_ref) || (vs != 0.f && vs * 256.f < v_ref));
      k_alike = k_alike || apart;
      v_alike = v_alike || apart;
    }
    const __half2 kr0 = __float2half2_rn(__shfl_sync(0xffffffffu, ks, 2 * pw) * k_inv), kr1 = __float2half2_rn(__shfl_sync(0xffffffffu, ks, 2 * pw + 1) * k_inv);
    const __half2 vr0 = __float2half2_rn(__shfl_sync(0xffffffffu, vs, 2 * pw) * v_inv), vr1 = __float2half2_rn(__shfl_sync(0xffffffffu, vs, 2 * pw + 1) * v_inv);
    if (pw == 0 && __any_sync(0xffffffffu, inside && page < 0) && lane == 0) kv_report(kv, HB_CACHE_BAD_PAGE);

    if (!mbar_wait_warp(&s.kv_empty[slot], phase, ctx, kRolePagedProducer)) return;
    if (pw == 0) {
      if (apart && lane < 8) s.group[at][lane] = make_float2(ks, vs);
      __syncwarp();
      if (lane == 0) {
        s.meta[at] = make_float4(k_ref, v_ref, __uint_as_float(gone), apart ? 1.f : 0.f);
        mbar_arrive(&s.meta_full[at]);
      }
    }
    store(slot, wk, k_alike, kr0, kr1);
    advance();
    if (j + 1 < nmax) fetch(k_base, kv.k_sp, kv.k_ss, j + 1, next, wk);
    ks = scale_of(kv.k_scale, next);
    vs = scale_of(kv.v_scale, next);
    if (!mbar_wait_warp(&s.kv_empty[slot], phase, ctx, kRolePagedProducer)) return;
    store(slot, wv, v_alike, vr0, vr1);
    advance();
    page = next;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPagedTilesThreads, 1) fa_paged_tiles_kernel(const __grid_constant__ FaPagedTilesParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  using Smem = FaPagedTilesSmem<D>;
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  AbortCtx ctx{&s.abort_flag, p.status};
  if (threadIdx.x == 0) {
    s.abort_flag = 0;
    s.found = -1;
    s.descends = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 4);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.o_full[i], 1);
    }
    for (int i = 0; i < Smem::kStages; ++i) {
      mbar_init(&s.kv_full[i], 4);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < Smem::kMeta; ++i) mbar_init(&s.meta_full[i], 1);
    mbar_init(&s.drain, 1);
    fence_mbar_init();
    if ((smem_u32(smem_raw) & 1023u) != 0u) raise_abort(ctx, kStatusSmemMisaligned);
  }
  __syncthreads();
  // For the rows kernel of the call too, where there is one.  Beside that, let in behind its wait and waiting at the end, D64 batches of prompts and
  // single tokens took 89.8 us instead of 93.9, D128 ones 108.2 instead of 107.4; but what is earlier is visible only behind a wait of one's own.
  grid_wait();

  // ---- the block's item: the last 256 rows (which see most keys) of every KV head first, where sequences are alike of all of
  // them; sequences in order elsewhere
  PagedItem it;
  {
    const KvView& kv = p.c;
    const int index = p.splits == 1 ? blockIdx.x : blockIdx.x / p.splits;  // of the item
    const int split = static_cast<int>(blockIdx.x) - index * p.splits;
    long long before = 0;
    if (kv.starts == nullptr && threadIdx.x == 0) {
      s.found = 0;
      s.found_at = 0;
    }
    for (int b0 = kv.starts == nullptr ? kv.B : 0; b0 < kv.B; b0 += kPagedTilesThreads) {
      const int b = b0 + threadIdx.x;
      const long long own = b < kv.B ? static_cast<long long>(paged_blocks_of(p, kv_seq(kv, b))) * kv.Hkv : 0;
      if (b < kv.B && kv_start(kv, b) > kv_start(kv, b + 1)) s.descends = 1;  // see kv_descends
      long long upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      if (b0 > 0) __syncthreads();
      if (lane == 31) s.sums[warp] = upto;
      __syncthreads();
      upto += before;
      for (int w = 0; w < kPagedTilesThreads / 32; ++w) {
        if (w < warp) upto += s.sums[w];
        before += s.sums[w];
      }
      if (upto > index && upto - own <= index) {
        s.found = b;
        s.found_at = upto - own;
      }
    }
    if (blockIdx.x == 0) {
      for (int b = threadIdx.x; b < kv.B; b += kPagedTilesThreads) {
        const uint32_t f = kv_seq_faults(kv, b);
        if (f != 0) kv_report(kv, f);
      }
    }
    __syncthreads();
    if (s.found < 0 || s.descends != 0) {  // the grid is cut for the most items that so many rows can be
      if (p.splits > 1 && split == 0 && threadIdx.x == 0) p.parts[index].count = 0;
      return;
    }
    it.b = s.found;
    const int in = static_cast<int>(index - s.found_at);
    int rank = fast_div(in, p.by_hkv);
    it.h = in - rank * kv.Hkv;
    if (kv.starts == nullptr) {
      const int turn = fast_div(rank, p.by_b);
      it.b = rank - turn * kv.B;
      rank = turn;
    }
    it.s = kv_seq(kv, it.b);
    it.rows = it.s.n * p.group;
    it.row0 = (paged_blocks_of(p, it.s) - 1 - rank) * kPagedBlockRows;
    const int tiles = max((it.s.len + kTileN - 1) / kTileN, 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r0 = it.row0 + kTileM * i;
      if (r0 >= it.rows) {
        it.n[i] = 0;
      } else if (p.causal) {
        const int last = it.s.pos0() + fast_div(min(r0 + kTileM, it.rows) - 1, p.by_group);  // position of the last row
        it.n[i] = max(min(tiles, last / kTileN + 1), 1);
      } else {
        it.n[i] = tiles;
      }
    }
    // its key tiles in equal parts, of four at least
    const int most = max(it.n[0], it.n[1]), parts = min(p.splits, (most + 3) / 4);
    it.whole = parts == 1;
    if (p.splits > 1 && split == 0 && threadIdx.x == 0) {
      PagedParts x;
      x.count = parts;
      x.h = it.h;
      x.row0 = it.row0;
      x.rows = it.rows;
      x.start = it.s.start;
      p.parts[index] = x;
    }
    if (split >= parts) return;
    it.j0 = it.whole ? 0 : static_cast<int>(static_cast<unsigned>(most) * split / parts);  // most < 2^24, parts at most 16
    it.j1 = it.whole ? most : static_cast<int>(static_cast<unsigned>(most) * (split + 1) / parts);
    it.n[0] = min(it.n[0], it.j1);
    it.n[1] = min(it.n[1], it.j1);
  }

  if (warp < 8) {
    paged_copy_queries<T, D>(p, s, it, warp >> 2);
    cp_async_commit();
  } else if (warp == 8) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(s.tmem_base);
  const bool run = s.abort_flag == 0;
  // 512 threads start with 128 registers each: four warps return 80, four 16, eight grow by 48
  static_assert(8 * 32 * (176 - 128) <= 4 * 32 * (128 - 48) + 4 * 32 * (128 - 112), "setmaxnreg budget does not balance");
  if (warp < 8) {
    reg_inc<176>();
    if (run) paged_softmax_role<T, D>(p, s, ctx, tmem, it, warp >> 2);
  } else if (warp < 12) {
    reg_dec<48>();
    if (run && warp == 8) {
      paged_mma_role<D>(s, ctx, tmem, it);
      __syncwarp();
      if (s.abort_flag && lane == 0) {
        umma_commit(&s.drain);  // aborting: let the tensor pipe drain before TMEM is released
        mbar_wait(&s.drain, 0, ctx, kRolePagedDrain);
      }
    }
  } else {
    reg_dec<112>();
    if (run) paged_producer_role<D>(p, s, ctx, it, warp - 12);
  }
  __syncwarp();
  cp_async_wait<0>();
  tc_fence_before();
  grid_launch_dependents();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merges the parts of the items that are in any: a block has 32 rows of an item, a warp four of them, a lane D / 32 columns.
template <typename T, int D>
__global__ void __launch_bounds__(256) fa_paged_tiles_combine_kernel(const __grid_constant__ FaPagedTilesParams p) {
  grid_launch_dependents();
  grid_wait();
  constexpr int kCols = D / 32, kBlocks = kPagedBlockRows / 32;
  const long long item = blockIdx.x / kBlocks;
  const PagedParts x = p.parts[item];
  if (x.count < 2) return;
  const int lane = threadIdx.x & 31, r0 = static_cast<int>(blockIdx.x - item * kBlocks) * 32 + (threadIdx.x >> 5) * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + k, row = x.row0 + r;
    if (row >= x.rows) return;
    auto at = [&](int part) -> long long { return (item * p.splits + part) * kPagedBlockRows + r; };
    float top = lane < x.count ? p.part_lse[at(lane)] : -INFINITY;  // at most 32 parts
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
    float acc[kCols] = {}, sum = 0.f;
    for (int part = 0; part < x.count; ++part) {
      const float lse = p.part_lse[at(part)];
      if (lse == -INFINITY) continue;  // nothing was written
      const float wt = fast_exp2(lse - top);
      const float* src = p.part_o + at(part) * D + lane * kCols;
      sum += wt;
      if constexpr (kCols == 4) {
        const float4 y = *reinterpret_cast<const float4*>(src);
        acc[0] = fmaf(wt, y.x, acc[0]);
        acc[1] = fmaf(wt, y.y, acc[1]);
        acc[2] = fmaf(wt, y.z, acc[2]);
        acc[3] = fmaf(wt, y.w, acc[3]);
      } else {
        const float2 y = *reinterpret_cast<const float2*>(src);
        acc[0] = fmaf(wt, y.x, acc[0]);
        acc[1] = fmaf(wt, y.y, acc[1]);
      }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    const int tok = fast_div(row, p.by_group), head = x.h * p.group + row - tok * p.group;
    T* dst = static_cast<T*>(p.o) + static_cast<long long>(x.start + tok) * p.o_st + head * p.o_sh + lane * kCols;
    if constexpr (kCols == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(Pack2<T>::pack(acc[0] * inv, acc[1] * inv), Pack2<T>::pack(acc[2] * inv, acc[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = Pack2<T>::pack(acc[0] * inv, acc[1] * inv);
    if (lane == 0 && p.lse != nullptr)
      p.lse[static_cast<long long>(x.start + tok) * p.Hq + head] = (sum != 0.f ? top + fast_log2(sum) : -INFINITY) * 0.6931471805599453f;
  }
}

}  // namespace hb
