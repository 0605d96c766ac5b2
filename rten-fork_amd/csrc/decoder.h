// Shared parts of the decoder operators (rotary.hip, paged_attention.hip,
// sampling.hip): the paged cache and the sequences of a call as the kernels
// see them, and the checks of their C descriptors.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "ctx.h"
#include "fastdiv_dev.h"

namespace rtenhip {

typedef unsigned long long u64;

// ---- sums over a wave ------------------------------------------------------------------

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp(u64 x) {
  return (u64)dpp<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)x);
}
// Inclusive prefix over the rows of 16 lanes, the halves and the whole of a wave,
// all of whose lanes are active: shifts within rows, then the last lanes of rows.
template <typename T>
__device__ __forceinline__ T row_scan(T x) {
  x += dpp<0x111, 0xf>(x);
  x += dpp<0x112, 0xf>(x);
  x += dpp<0x114, 0xf>(x);
  x += dpp<0x118, 0xf>(x);
  return x;
}
template <typename T>
__device__ __forceinline__ T half_scan(T x) {
  x = row_scan(x);
  x += dpp<0x142, 0xa>(x);
  return x;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  x = half_scan(x);
  x += dpp<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ u64 lane_of(u64 x, int lane) {
  return (u64)lane_of((uint32_t)(x >> 32), lane) << 32 | lane_of((uint32_t)x, lane);
}
template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
  return lane_of(wave_scan(x), 63);
}

// ---- descriptors -----------------------------------------------------------------------

// A paged cache for the kernels: element strides, any order of page, slot and
// head, head_dim contiguous elements per row.
struct CacheView {
  char *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int64_t n_pages;
  FastDiv page_div;
  int page_size, heads, dim;
};

struct SeqView {
  const int* table;     // [n][max_pages], row stride table_stride
  int64_t table_stride;
  const int* kv_lens;   // [n]: cached tokens, the call's new ones included
  const int* q_starts;  // [n + 1], or null: one new token per sequence
  int n, max_pages, tokens;
};

// The first new token of sequence s (q_starts as given may hold anything: the
// kernels only ever use values brought into [0, tokens]).
__device__ __forceinline__ int seq_start(const SeqView& v, int s) {
  if (!v.q_starts) return s < v.tokens ? s : v.tokens;
  const int a = v.q_starts[s];
  return a < 0 ? 0 : a > v.tokens ? v.tokens : a;
}

// The entry for token `tok` in the page row `row`, -1 past the table.  What it
// is is looked at only where it is needed (page_ok): a check right behind the
// load would wait for it, and for every load before it.
__device__ __forceinline__ int page_entry(const int* row, int max_pages, const CacheView& c, int tok) {
  const int at = fdiv(tok, c.page_div);
  return at < max_pages ? row[at] : -1;
}
__device__ __forceinline__ bool page_ok(const CacheView& c, int page) {
  return (unsigned)page < (uint64_t)c.n_pages;
}

rtenhip_status cache_view(const rtenhip_kv_cache* cache, CacheView& v, int& dtype);
rtenhip_status seq_view(const rtenhip_sequences* seqs, int64_t tokens, SeqView& v);
// q / k / v / out rows [tokens, heads, dim]: f32, unit stride along dim, rows
// on 16 bytes.
rtenhip_status check_rows(const rtenhip_tensor* t, int64_t tokens, int64_t heads, int64_t dim, const char* shape_msg,
                          const char* align_msg);
// Whether two views of [tokens, heads, dim] rows share memory without being
// the same view.
bool rows_clash(const rtenhip_tensor* a, const rtenhip_tensor* b);

// Whether rows of `dim` elements at these strides, the extents n, are all apart
// (what is written must not be written twice).
bool rows_apart(const int64_t* n, const int64_t* strides, int count, int64_t dim);

// A launch has fewer than 2^32 threads.
inline bool launchable(int64_t blocks, int64_t threads) { return blocks * threads <= int64_t(UINT32_MAX); }

// Makes the context's device current for a launch and puts back the caller's.
struct DeviceScope {
  int before = -1;
  rtenhip_status status = RTENHIP_OK;
  explicit DeviceScope(int device) {
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before == device) before = -1;
    else if (e == hipSuccess) e = hipSetDevice(device);
    if (e != hipSuccess) status = hip_fail(e, "hipSetDevice");
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

}  // namespace rtenhip
