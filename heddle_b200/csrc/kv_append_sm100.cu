// hb_kv_append: new keys (rotated by their positions) and values into the pages of the cache as e4m3 codes, and the queries of the
// same tokens rotated beside them.
//
// A unit of work is what a call writes of one page for one KV head: keys and values of up to page_size tokens.  A group of
// threads (a warp for single tokens, a whole block for prompts) owns the unit, so that the largest magnitude, the page's scale and the
// codes need no other exchange: it goes over its tokens once for the maximum and once for the codes, the second time out of L1.
// Scales are powers of two: dividing by one is exact, and so is turning an earlier code over to a larger scale but for the bits
// that fall below e4m3's smallest step.  They grow only where a new token needs it, so that a decode step nearly always writes its
// own 2 D bytes and leaves the page alone.
//
// What bounds it: HBM.  Four prompts of 2048 tokens with their queries (Hq32 Hkv8 D128 bf16, 189 MB) 37.4 us in a captured graph, 5.0 TB/s; one token for 64 sequences 3.5 us,
// a launch and a chain of four loads.
#include "host_common.h"
#include "fast_div.h"
#include "kv_cache.h"
#include "ptx_sm100.cuh"

#include <algorithm>

namespace hb {

struct KvAppendParams {
  KvView c;
  const void* k;
  const void* v;
  const void* q;
  void* q_out;
  long long k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh;
  const float* cos;
  const float* sin;
  int rope_len;
  int blocks_each;   // without starts: page blocks of a sequence
  int units;         // of the cache
  int cache_blocks;  // blocks of the grid that write the cache; those behind rotate queries
  FastDiv by_hkv, by_q_row, by_each;
  int q_items;
};

constexpr int kAppendThreads = 256;
constexpr int kMinScaleExp = -100, kMaxScaleExp = 119;  // a code times the scale is a normal bf16, and finite

__device__ __forceinline__ float append_pow2(int e) { return __int_as_float((e + 127) << 23); }

// The smallest exponent e with a <= 448 * 2^e; a is finite, not negative.
__device__ __forceinline__ int append_exponent(float a) {
  if (!(a > 0.f)) return kMinScaleExp;
  const int bits = __float_as_int(a);
  int e = (bits >> 23) - 127, frac = bits & 0x7fffff;  // a = 1.frac * 2^e; 448 = 1.75 * 2^8
  if (bits < 0x800000) return kMinScaleExp;             // subnormal
  e = e - 8 + (frac > 0x600000 ? 1 : 0);
  return min(max(e, kMinScaleExp), kMaxScaleExp);
}

template <typename T>
__device__ __forceinline__ void append_unpack8(const uint4& w, float* f) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) Pack2<T>::unpack(u[i], f[2 * i], f[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ void append_load8(const T* p, float* f) {
  append_unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
}
template <typename T>
__device__ __forceinline__ void append_store8(T* p, const float* f) {
  uint4 w;
  w.x = Pack2<T>::pack(f[0], f[1]);
  w.y = Pack2<T>::pack(f[2], f[3]);
  w.z = Pack2<T>::pack(f[4], f[5]);
  w.w = Pack2<T>::pack(f[6], f[7]);
  *reinterpret_cast<uint4*>(p) = w;
}
// lo and hi: the pairs x_i, x_{i + D/2}; every product and sum is rounded by itself
__device__ __forceinline__ void append_rotate(float* lo, float* hi, const float* cos, const float* sin) {
  const float4 c0 = reinterpret_cast<const float4*>(cos)[0], c1 = reinterpret_cast<const float4*>(cos)[1];
  const float4 s0 = reinterpret_cast<const float4*>(sin)[0], s1 = reinterpret_cast<const float4*>(sin)[1];
  const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = lo[i], b = hi[i];
    lo[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    hi[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}
__device__ __forceinline__ uint32_t append_codes4(const float* f, float inv) {
  uint16_t a, b;  // the first source is the upper byte
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(f[1] * inv), "f"(f[0] * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(f[3] * inv), "f"(f[2] * inv));
  return a | (static_cast<uint32_t>(b) << 16);
}
// Two codes times a power of two of at most 1, rounded again.  In fp16 the product is exact down to 2^-24, far below half of e4m3's
// smallest step (2^-10), and a factor that fp16 cannot hold takes every code there.
__device__ __forceinline__ uint32_t append_shrink(uint32_t codes, __half2 factor) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t c = static_cast<uint16_t>(codes >> (16 * i));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&h), factor);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
    out |= static_cast<uint32_t>(r) << (16 * i);
  }
  return out;
}

// The sequence of row t: the last b with starts[b] <= t.
__device__ __forceinline__ int append_seq_of(const KvAppendParams& p, int t) {
  if (p.c.starts == nullptr) return fast_div(t, p.by_each);
  int lo = 0, hi = p.c.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (kv_start(p.c, mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Rotates the queries: a thread has eight pairs of kQueryRows rows, whose loads are on their way together.
constexpr int kQueryRows = 2;
template <typename T, int D>
__device__ __forceinline__ void append_queries(const KvAppendParams& p) {
  constexpr int kPieces = D / 16;
  const int item0 = (static_cast<int>(blockIdx.x) - p.cache_blocks) * kAppendThreads * kQueryRows + static_cast<int>(threadIdx.x);
  uint4 lo4[kQueryRows], hi4[kQueryRows];
  int pos[kQueryRows];  // -1: nothing to do
  T* dst[kQueryRows];
#pragma unroll
  for (int k = 0; k < kQueryRows; ++k) {
    const int item = item0 + k * kAppendThreads;
    pos[k] = -1;
    if (item >= p.q_items) continue;
    const int t = fast_div(item, p.by_q_row), r = item - t * static_cast<int>(p.by_q_row.d);
    const int head = r / kPieces, piece = r % kPieces;
    const T* src = static_cast<const T*>(p.q) + t * p.q_st + head * p.q_sh + piece * 8;
    lo4[k] = *reinterpret_cast<const uint4*>(src);
    hi4[k] = *reinterpret_cast<const uint4*>(src + D / 2);
    dst[k] = static_cast<T*>(p.q_out) + t * p.qo_st + head * p.qo_sh + piece * 8;
    const int b = append_seq_of(p, t);
    const KvSeq s = kv_seq(p.c, b);
    const int at = t - s.start, x = kv_append_position(p.c, b, s) + at;
    // not a row of no sequence, nor one behind the tables (reported with the keys)
    if (at >= 0 && at < s.n && (p.cos == nullptr || (x >= 0 && x < p.rope_len))) pos[k] = max(x, 0);
  }
  const int piece = item0 % kPieces;  // of every row of the thread
#pragma unroll
  for (int k = 0; k < kQueryRows; ++k) {
    if (pos[k] < 0) continue;
    if (p.cos != nullptr) {
      float lo[8], hi[8];
      append_unpack8<T>(lo4[k], lo);
      append_unpack8<T>(hi4[k], hi);
      const long long at = static_cast<long long>(pos[k]) * (D / 2) + piece * 8;
      append_rotate(lo, hi, p.cos + at, p.sin + at);
      append_store8(dst[k], lo);
      append_store8(dst[k] + D / 2, hi);
    } else {
      *reinterpret_cast<uint4*>(dst[k]) = lo4[k];
      *reinterpret_cast<uint4*>(dst[k] + D / 2) = hi4[k];
    }
  }
}

// GS threads own a unit.
template <typename T, int D, int GS>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const __grid_constant__ KvAppendParams p) {
  grid_wait();
  if (p.c.starts != nullptr && __syncthreads_or(kv_descends(p.c))) {
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b < p.c.B; b += kAppendThreads) {
        const uint32_t f = kv_seq_faults(p.c, b);
        if (f != 0) kv_report(p.c, f);
      }
    return;
  }
  if (static_cast<int>(blockIdx.x) >= p.cache_blocks) {
    append_queries<T, D>(p);
    return;
  }
  constexpr int kPieces = D / 16;  // a token's threads: eight pairs of its key, sixteen elements of its value each
  __shared__ float s_max[2][kAppendThreads / 32];
  const KvView& c = p.c;
  const int group = threadIdx.x / GS, tid = threadIdx.x % GS;
  const int unit = static_cast<int>(blockIdx.x) * (kAppendThreads / GS) + group;
  if (unit >= p.units) return;
  const int slot = fast_div(unit, p.by_hkv), h = unit - slot * c.Hkv;
  int b, block;
  if (c.starts == nullptr) {
    b = slot / p.blocks_each;
    block = slot - b * p.blocks_each;
  } else {
    // sequence b has the slots from starts[b] / page_size + 2 b on: n rows lie in at most (n - 1) / page_size + 2 pages
    int lo = 0, hi = c.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((kv_start(c, mid) >> c.page_shift) + 2 * mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    block = slot - ((kv_start(c, b) >> c.page_shift) + 2 * b);
  }
  const KvSeq s = kv_seq(c, b);
  const int pos0 = kv_append_position(c, b, s);
  if (h == 0 && block == 0 && tid == 0) {
    uint32_t f = kv_seq_faults(c, b);
    if (p.cos != nullptr && s.n > 0 && pos0 + s.n > p.rope_len) f |= HB_CACHE_BAD_POSITION;
    if (f != 0) kv_report(c, f);
  }
  const int limit = p.cos != nullptr ? min(s.len, p.rope_len) : s.len;  // tokens behind the tables, of pages or of angles, are not written
  block += max(pos0, 0) >> c.page_shift;
  if (block < 0 || block >= c.max_pages) return;
  const int begin = block << c.page_shift;
  const int low = max(pos0, begin), high = min(limit, begin + (1 << c.page_shift));
  if (s.n == 0 || low >= high) return;
  const int page = kv_page(c, b, block);
  if (page < 0) {
    if (tid == 0) kv_report(c, HB_CACHE_BAD_PAGE);
    return;
  }
  const int earlier = low - begin, total = (high - low) * kPieces;
  const T* k = static_cast<const T*>(p.k) + h * p.k_sh;
  const T* v = static_cast<const T*>(p.v) + h * p.v_sh;
  const int piece = tid % kPieces;

  // one token's pairs and elements of this thread; false where its key or value (over all its threads) is not finite
  auto load = [&](int i, bool live, float (&x)[16], float (&y)[16]) -> bool {
    bool finite = true;
    if (live) {
      const int pos = low + i / kPieces;
      const long long row = s.start + (pos - pos0);
      const T* kr = k + row * p.k_st + piece * 8;
      const T* vr = v + row * p.v_st + piece * 16;
      append_load8(kr, x);
      append_load8(kr + D / 2, x + 8);
      append_load8(vr, y);
      append_load8(vr + 8, y + 8);
      if (p.cos != nullptr)
        append_rotate(x, x + 8, p.cos + static_cast<long long>(pos) * (D / 2) + piece * 8, p.sin + static_cast<long long>(pos) * (D / 2) + piece * 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) finite = finite && fabsf(x[e]) <= 3.402823466e38f && fabsf(y[e]) <= 3.402823466e38f;
    }
    const unsigned votes = __ballot_sync(0xffffffffu, finite);
    const int first = (threadIdx.x & 31) / kPieces * kPieces;
    return ((votes >> first) & ((1u << kPieces) - 1u)) == ((1u << kPieces) - 1u);
  };

  float k_max = 0.f, v_max = 0.f;
  for (int i0 = 0; i0 < total; i0 += GS) {
    float x[16], y[16];
    const bool live = i0 + tid < total;
    if (load(i0 + tid, live, x, y) && live) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        k_max = fmaxf(k_max, fabsf(x[e]));
        v_max = fmaxf(v_max, fabsf(y[e]));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    k_max = fmaxf(k_max, __shfl_xor_sync(0xffffffffu, k_max, o));
    v_max = fmaxf(v_max, __shfl_xor_sync(0xffffffffu, v_max, o));
  }
  const long long scale_at = static_cast<long long>(page) * c.Hkv + h;
  float k_old = 0.f, v_old = 0.f;
  if (earlier > 0) {
    k_old = c.k_scale[scale_at];
    v_old = c.v_scale[scale_at];
  }
  if constexpr (GS > 32) {
    constexpr int kWarps = GS / 32;
    if ((tid & 31) == 0) {
      s_max[0][threadIdx.x >> 5] = k_max;
      s_max[1][threadIdx.x >> 5] = v_max;
    }
    if constexpr (GS == kAppendThreads) __syncthreads();
    else named_bar_sync(1 + group, GS);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      k_max = fmaxf(k_max, s_max[0][group * kWarps + w]);
      v_max = fmaxf(v_max, s_max[1][group * kWarps + w]);
    }
  } else {
    __syncwarp();
  }
  // every thread of the group has read the old scales
  const int ek = append_exponent(k_max), ev = append_exponent(v_max);
  const float k_new = fmaxf(append_pow2(ek), k_old), v_new = fmaxf(append_pow2(ev), v_old);
  const float k_inv = 1.f / k_new, v_inv = 1.f / v_new;
  if (tid == 0) {
    c.k_scale[scale_at] = k_new;
    c.v_scale[scale_at] = v_new;
  }
  uint8_t* kp = c.k + kv_offset(page, c.k_sp) + kv_offset(h, c.k_sh);
  uint8_t* vp = c.v + kv_offset(page, c.v_sp) + kv_offset(h, c.v_sh);
  auto shrink = [&](uint8_t* base, unsigned stride, float factor) {
    const __half2 f = __float2half2_rn(factor);
    for (int i = tid; i < earlier * kPieces; i += GS) {
      uint4* at = reinterpret_cast<uint4*>(base + kv_offset(i / kPieces, stride) + piece * 16);
      uint4 w = *at;
      w.x = append_shrink(w.x, f);
      w.y = append_shrink(w.y, f);
      w.z = append_shrink(w.z, f);
      w.w = append_shrink(w.w, f);
      *at = w;
    }
  };
  if (earlier > 0 && k_new > k_old) shrink(kp, c.k_ss, k_old / k_new);
  if (earlier > 0 && v_new > v_old) shrink(vp, c.v_ss, v_old / v_new);
  for (int i0 = 0; i0 < total; i0 += GS) {
    float x[16], y[16];
    const bool live = i0 + tid < total;
    const bool finite = load(i0 + tid, live, x, y);
    if (!live) continue;
    const int place = earlier + (i0 + tid) / kPieces;
    uint2 lo = make_uint2(append_codes4(x, k_inv), append_codes4(x + 4, k_inv));
    uint2 hi = make_uint2(append_codes4(x + 8, k_inv), append_codes4(x + 12, k_inv));
    uint4 val = make_uint4(append_codes4(y, v_inv), append_codes4(y + 4, v_inv), append_codes4(y + 8, v_inv), append_codes4(y + 12, v_inv));
    if (!finite) {
      lo = hi = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      val = make_uint4(0u, 0u, 0u, 0u);
    }
    *reinterpret_cast<uint2*>(kp + kv_offset(place, c.k_ss) + piece * 8) = lo;
    *reinterpret_cast<uint2*>(kp + kv_offset(place, c.k_ss) + D / 2 + piece * 8) = hi;
    *reinterpret_cast<uint4*>(vp + kv_offset(place, c.v_ss) + piece * 16) = val;
  }
  grid_launch_dependents();  // let in at the start, they take the slots of blocks that have not begun: B4 prompts 37.3 -> 37.7 us
}

template <typename T, int D>
static cudaError_t append_launch(const KvAppendParams& p, int gs, unsigned grid, cudaStream_t stream) {
  if (gs == 32) return launch_dependent(kv_append_kernel<T, D, 32>, grid, kAppendThreads, 0, stream, 0, p);
  if (gs == 64) return launch_dependent(kv_append_kernel<T, D, 64>, grid, kAppendThreads, 0, stream, 0, p);
  return launch_dependent(kv_append_kernel<T, D, kAppendThreads>, grid, kAppendThreads, 0, stream, 0, p);
}

}  // namespace hb

extern "C" int hb_kv_append(const hb_kv_append_args* a) {
  using namespace hb;
  clear_error();
  const char* fn = "hb_kv_append";
  if (a == nullptr) return set_error(HB_ERR_BAD_ARG, "%s: args is NULL", fn);
  const hb_kv_cache& c = a->cache;
  bool empty = false;
  int rc = kv_cache_check(fn, c, &empty);
  if (rc != HB_OK) return rc;
  if (a->dtype != HB_BF16 && a->dtype != HB_FP16) return set_error(HB_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are built)", fn, a->dtype);
  if ((a->rope_cos == nullptr) != (a->rope_sin == nullptr) || a->rope_len < 0)
    return set_error(HB_ERR_BAD_ARG, "%s: rope_cos and rope_sin come together, rope_len may not be negative", fn);
  if (a->q != nullptr && a->Hq <= 0) return set_error(HB_ERR_BAD_ARG, "%s: Hq must be positive where q is given", fn);
  if (empty) return HB_OK;
  if (a->k == nullptr || a->v == nullptr || (a->q != nullptr && a->q_out == nullptr)) return set_error(HB_ERR_BAD_ARG, "%s: NULL pointer", fn);
  uint64_t bits = reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->rope_cos) |
                  reinterpret_cast<uintptr_t>(a->rope_sin) |
                  static_cast<uint64_t>(2 * (a->k_stride_t | a->k_stride_h | a->v_stride_t | a->v_stride_h));
  if (a->q != nullptr)
    bits |= reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out) |
            static_cast<uint64_t>(2 * (a->q_stride_t | a->q_stride_h | a->qo_stride_t | a->qo_stride_h));
  if ((bits & 15u) != 0) return set_error(HB_ERR_ALIGN, "%s: rows of k, v, q and the rotary tables must be 16-byte aligned", fn);
  const int pieces = c.D / 16;
  const int64_t q_items = a->q != nullptr ? static_cast<int64_t>(c.T) * a->Hq * pieces : 0;
  int64_t each = 0, slots;
  if (c.starts == nullptr) {
    each = c.T / c.B == 1 ? 1 : (c.T / c.B - 1) / c.page_size + 2;
    slots = each * c.B;
  } else {
    slots = static_cast<int64_t>(c.T) / c.page_size + 2ll * c.B;
  }
  const int64_t units = slots * c.Hkv;
  if (q_items > 0x7fff0000ll || units > 0x7fff0000ll)
    return set_error(HB_ERR_UNSUPPORTED, "%s: more than 2^31 pieces of work (T = %d, B = %d)", fn, c.T, c.B);
  DeviceState* st = nullptr;
  rc = get_device_state(&st);
  if (rc != HB_OK) return rc;
  KvAppendParams p;
  p.c = kv_view(c, st);
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.q_out = a->q_out;
  p.k_st = a->k_stride_t;
  p.k_sh = a->k_stride_h;
  p.v_st = a->v_stride_t;
  p.v_sh = a->v_stride_h;
  p.q_st = a->q_stride_t;
  p.q_sh = a->q_stride_h;
  p.qo_st = a->qo_stride_t;
  p.qo_sh = a->qo_stride_h;
  p.cos = a->rope_cos;
  p.sin = a->rope_sin;
  p.rope_len = a->rope_len;
  p.blocks_each = static_cast<int>(each);
  p.units = static_cast<int>(units);
  p.by_hkv = make_fast_div(c.Hkv);
  p.by_q_row = make_fast_div(a->q != nullptr ? a->Hq * pieces : 1);
  p.by_each = make_fast_div(p.c.each > 0 ? p.c.each : 1);
  p.q_items = static_cast<int>(q_items);
  // threads of a unit: two rounds over the tokens that a page takes on average
  const int64_t work = std::min<int64_t>(c.page_size, (static_cast<int64_t>(c.T) + c.B - 1) / c.B) * pieces;
  const int gs = work <= 64 ? 32 : work <= 128 ? 64 : kAppendThreads;
  p.cache_blocks = static_cast<int>((units + kAppendThreads / gs - 1) / (kAppendThreads / gs));
  const int64_t grid = p.cache_blocks + (q_items + kAppendThreads * kQueryRows - 1) / (kAppendThreads * kQueryRows);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  cudaError_t err;
  if (a->dtype == HB_BF16)
    err = c.D == 128 ? append_launch<__nv_bfloat16, 128>(p, gs, static_cast<unsigned>(grid), stream)
                     : append_launch<__nv_bfloat16, 64>(p, gs, static_cast<unsigned>(grid), stream);
  else
    err = c.D == 128 ? append_launch<__half, 128>(p, gs, static_cast<unsigned>(grid), stream)
                     : append_launch<__half, 64>(p, gs, static_cast<unsigned>(grid), stream);
  HB_CUDA_CHECK(err);
  return HB_OK;
}
