// The paged key/value cache as its kernels see it (hb_kv_cache in the C ABI): checks on the host, sequences and pages on the device.
#pragma once

#include <initializer_list>

#include "host_common.h"

namespace hb {

struct KvView {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  unsigned k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;  // strides of pages, heads and tokens
  const int* table;
  const int* lens;
  const int* starts;  // nullptr: `each` rows a sequence
  long long table_stride;
  int num_pages, page_shift, Hkv, max_pages, B, T, each;
  uint32_t* fault;
};

// Checks every field that the host can see.  `empty`: the call has no rows, and the device pointers were not looked at.
inline int kv_cache_check(const char* fn, const hb_kv_cache& c, bool* empty) {
  *empty = false;
  if (c.B < 0 || c.T < 0 || c.Hkv <= 0 || c.num_pages < 0 || c.max_pages < 0)
    return set_error(HB_ERR_BAD_ARG, "%s: B, T, num_pages and max_pages may not be negative, Hkv must be positive", fn);
  if (c.D != 64 && c.D != 128) return set_error(HB_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are built)", fn, c.D);
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
    return set_error(HB_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64 and 128 are built)", fn, c.page_size);
  if (static_cast<int64_t>(c.max_pages) * c.page_size > 0x7fffff00ll)
    return set_error(HB_ERR_UNSUPPORTED, "%s: max_pages * page_size exceeds 2^31", fn);
  if (c.B > 0 && c.starts == nullptr && c.T % c.B != 0)
    return set_error(HB_ERR_BAD_ARG, "%s: without starts, T = %d rows must be a multiple of B = %d", fn, c.T, c.B);
  if (c.B == 0 || c.T == 0) {
    *empty = true;
    return HB_OK;
  }
  if (c.page_table == nullptr || c.seq_lens == nullptr || c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr)
    return set_error(HB_ERR_BAD_ARG, "%s: NULL cache pointer", fn);
  for (int64_t s : {c.k_stride_p, c.k_stride_h, c.k_stride_s, c.v_stride_p, c.v_stride_h, c.v_stride_s})
    if (s < 0 || s > 0xffffffffll) return set_error(HB_ERR_UNSUPPORTED, "%s: strides of the pages must be within 0 .. 2^32 - 1", fn);
  const uintptr_t words = reinterpret_cast<uintptr_t>(c.page_table) | reinterpret_cast<uintptr_t>(c.seq_lens) |
                          reinterpret_cast<uintptr_t>(c.starts) | reinterpret_cast<uintptr_t>(c.k_scale) | reinterpret_cast<uintptr_t>(c.v_scale);
  const uint64_t rows = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | static_cast<uint64_t>(c.k_stride_p) |
                        static_cast<uint64_t>(c.k_stride_h) | static_cast<uint64_t>(c.k_stride_s) | static_cast<uint64_t>(c.v_stride_p) |
                        static_cast<uint64_t>(c.v_stride_h) | static_cast<uint64_t>(c.v_stride_s);
  if ((words & 3u) != 0 || (rows & 15u) != 0)
    return set_error(HB_ERR_ALIGN, "%s: rows of codes must be 16-byte aligned, table, lengths, starts and scales 4-byte aligned", fn);
  return HB_OK;
}

inline KvView kv_view(const hb_kv_cache& c, const DeviceState* st) {
  KvView v;
  v.k = static_cast<uint8_t*>(c.k);
  v.v = static_cast<uint8_t*>(c.v);
  v.k_scale = c.k_scale;
  v.v_scale = c.v_scale;
  v.k_sp = static_cast<unsigned>(c.k_stride_p);
  v.k_sh = static_cast<unsigned>(c.k_stride_h);
  v.k_ss = static_cast<unsigned>(c.k_stride_s);
  v.v_sp = static_cast<unsigned>(c.v_stride_p);
  v.v_sh = static_cast<unsigned>(c.v_stride_h);
  v.v_ss = static_cast<unsigned>(c.v_stride_s);
  v.table = c.page_table;
  v.lens = c.seq_lens;
  v.starts = c.starts;
  v.table_stride = c.table_stride;
  v.num_pages = c.num_pages;
  v.page_shift = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
  v.Hkv = c.Hkv;
  v.max_pages = c.max_pages;
  v.B = c.B;
  v.T = c.T;
  v.each = c.starts == nullptr ? c.T / c.B : 0;
  v.fault = st->cache_fault;
  return v;
}

#ifdef __CUDACC__
__device__ __forceinline__ long long kv_offset(int n, unsigned stride) {  // n >= 0: one multiplication
  return static_cast<long long>(static_cast<unsigned long long>(static_cast<unsigned>(n)) * stride);
}
struct KvSeq {
  int start, n;  // its rows of the call
  int len;       // its tokens, those rows included
  __device__ __forceinline__ int pos0() const { return len - n; }  // position of its first row
};

// Row b of starts, within [0, T].
__device__ __forceinline__ int kv_start(const KvView& c, int b) {
  return c.starts == nullptr ? b * c.each : min(max(c.starts[b], 0), c.T);
}
__device__ __forceinline__ KvSeq kv_seq(const KvView& c, int b) {
  KvSeq s;
  s.start = kv_start(c, b);
  s.n = max(kv_start(c, b + 1) - s.start, 0);
  s.len = min(max(c.lens[b], 0), c.max_pages << c.page_shift);
  return s;
}
// The position that the sequence's first row is appended at: a length behind the page table's end moves no token in front of it.
__device__ __forceinline__ int kv_append_position(const KvView& c, int b, const KvSeq& s) { return max(c.lens[b], 0) - s.n; }
// Whether starts descend somewhere, of what this thread of a block looks at; the threads together look at all of them.  A call whose starts do
// has rows that belong to two sequences: it reports that and writes nothing.
__device__ __forceinline__ bool kv_descends(const KvView& c) {
  bool down = false;
  if (c.starts != nullptr)
    for (int b = threadIdx.x; b < c.B; b += blockDim.x) down = down || kv_start(c, b) > kv_start(c, b + 1);
  return down;
}
// What of sequence b kv_seq had to mend.
__device__ __forceinline__ uint32_t kv_seq_faults(const KvView& c, int b) {
  const KvSeq s = kv_seq(c, b);
  uint32_t f = (c.lens[b] != s.len || s.n > s.len) ? HB_CACHE_BAD_LENGTH : 0u;
  if (c.starts != nullptr && (c.starts[b] != s.start || c.starts[b + 1] != s.start + s.n)) f |= HB_CACHE_BAD_STARTS;
  return f;
}
// The page of block `block` (< max_pages) of sequence b, -1 where the table holds none of the cache's.
__device__ __forceinline__ int kv_page(const KvView& c, int b, int block) {
  const int id = c.table[b * c.table_stride + block];
  return static_cast<unsigned>(id) < static_cast<unsigned>(c.num_pages) ? id : -1;
}
__device__ __forceinline__ void kv_report(const KvView& c, uint32_t faults) { atomicOr(c.fault, faults); }
#endif

}  // namespace hb
