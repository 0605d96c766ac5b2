// Norm of queries and keys for each head with the position rotation, and the
// append of keys and values to the paged cache, in one pass
// (rtenhip_qk_norm_rotary_f32, rtenhip_qk_norm_rotary_append_f32), and the
// descriptor checks shared by the decoder operators (decoder.h).
#include "decoder.h"

#include <cmath>

namespace rtenhip {

// ---- descriptor checks (host) ------------------------------------------------

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// |strides| * extents stays far inside int64, so no offset can overflow.
static bool stride_ok(int64_t s) { return s >= 0 && s < (int64_t(1) << 40); }

rtenhip_status cache_view(const rtenhip_kv_cache* c, CacheView& v, int& dtype) {
  if (!c) return fail(RTENHIP_MISSING_INPUTS, "Missing cache");
  if (c->dtype != RTENHIP_CACHE_F32 && c->dtype != RTENHIP_CACHE_F16 && c->dtype != RTENHIP_CACHE_BF16)
    return fail(RTENHIP_INCORRECT_INPUT_TYPE, "Cache must be float32, float16 or bfloat16");
  if (c->n_heads < 1 || c->n_pages < 0 || c->n_pages > INT32_MAX || c->page_size < 1 || c->page_size > 65536)
    return fail(RTENHIP_INVALID_VALUE, "Invalid cache size");
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
    return fail(RTENHIP_UNSUPPORTED_VALUE, "head_dim must be a multiple of 8 from 8 to 256");
  if (c->n_pages && (!c->k || !c->v)) return fail(RTENHIP_MISSING_INPUTS, "Missing cache");
  const int64_t per16 = c->dtype == RTENHIP_CACHE_F32 ? 4 : 8;
  const int64_t extent[3] = {c->n_pages, c->page_size, c->n_heads};
  if (!aligned16(c->k) || !aligned16(c->v))
    return fail(RTENHIP_UNSUPPORTED_VALUE, "Cache rows must start on 16 bytes");
  for (int i = 0; i < 3; i++)
    for (const int64_t s : {c->k_strides[i], c->v_strides[i]}) {
      if (extent[i] > 1 && s % per16) return fail(RTENHIP_UNSUPPORTED_VALUE, "Cache rows must start on 16 bytes");
      if (!stride_ok(s)) return fail(RTENHIP_UNSUPPORTED_VALUE, "Unsupported cache strides");
    }
  // (An extent of 1 is only ever indexed by 0, whatever its stride says.)
  const auto st = [&](const int64_t* s, int i) { return extent[i] > 1 ? s[i] : 0; };
  v.k = (char*)c->k;
  v.v = (char*)c->v;
  v.k_page = st(c->k_strides, 0);
  v.k_slot = st(c->k_strides, 1);
  v.k_head = st(c->k_strides, 2);
  v.v_page = st(c->v_strides, 0);
  v.v_slot = st(c->v_strides, 1);
  v.v_head = st(c->v_strides, 2);
  v.n_pages = c->n_pages;
  v.page_div = make_fastdiv((uint32_t)c->page_size);
  v.page_size = c->page_size;
  v.heads = c->n_heads;
  v.dim = c->head_dim;
  dtype = c->dtype;
  return RTENHIP_OK;
}

rtenhip_status seq_view(const rtenhip_sequences* s, int64_t tokens, SeqView& v) {
  if (!s) return fail(RTENHIP_MISSING_INPUTS, "Missing sequences");
  if (s->n_seqs < 0 || s->max_pages < 0 || s->table_stride < 0)
    return fail(RTENHIP_INVALID_VALUE, "Invalid sequences");
  if (!s->q_starts && s->n_seqs != tokens)
    return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Without q_starts there is one row per sequence");
  if (s->n_seqs && (!s->kv_lens || (s->max_pages && !s->page_table)))
    return fail(RTENHIP_MISSING_INPUTS, "Missing sequences");
  for (const void* p : {(const void*)s->page_table, (const void*)s->kv_lens, (const void*)s->q_starts})
    if ((uintptr_t)p % 4) return fail(RTENHIP_UNSUPPORTED_VALUE, "Sequence arrays must be on 4 bytes");
  v.table = s->page_table;
  v.table_stride = s->table_stride;
  v.kv_lens = s->kv_lens;
  v.q_starts = s->q_starts;
  v.n = s->n_seqs;
  v.max_pages = s->max_pages;
  v.tokens = (int)tokens;
  return RTENHIP_OK;
}

rtenhip_status check_rows(const rtenhip_tensor* t, int64_t tokens, int64_t heads, int64_t dim, const char* shape_msg,
                          const char* align_msg) {
  if (!t) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  if (t->ndim != 3 || t->shape[0] != tokens || t->shape[1] != heads || t->shape[2] != dim)
    return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, shape_msg);
  if (tokens * heads == 0) return RTENHIP_OK;
  if (!t->data) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  if (!aligned16(t->data) || (dim > 1 && t->strides[2] != 1) || (tokens > 1 && t->strides[0] % 4) ||
      (heads > 1 && t->strides[1] % 4) || !stride_ok(t->strides[0]) || !stride_ok(t->strides[1]))
    return fail(RTENHIP_UNSUPPORTED_VALUE, align_msg);
  return RTENHIP_OK;
}

bool rows_apart(const int64_t* n, const int64_t* strides, int count, int64_t dim) {
  // Every stride has to step over all that the smaller ones reach.
  int64_t reach = dim;
  bool used[4] = {};
  for (int round = 0; round < count; round++) {
    int at = -1;
    for (int i = 0; i < count; i++)
      if (!used[i] && (at < 0 || strides[i] < strides[at])) at = i;
    used[at] = true;
    if (n[at] == 0) return true;
    if (n[at] == 1) continue;
    if (strides[at] < reach) return false;
    reach += (n[at] - 1) * strides[at];
  }
  return true;
}

static void span(const rtenhip_tensor* t, uintptr_t& lo, uintptr_t& hi) {
  int64_t last = 0;
  for (int i = 0; i < t->ndim; i++) last += (t->shape[i] - 1) * t->strides[i];
  lo = (uintptr_t)t->data;
  hi = lo + (uintptr_t)(last + 1) * 4;
}

bool rows_clash(const rtenhip_tensor* a, const rtenhip_tensor* b) {
  if (numel(*a) == 0 || numel(*b) == 0) return false;
  uintptr_t al, ah, bl, bh;
  span(a, al, ah);
  span(b, bl, bh);
  if (ah <= bl || bh <= al) return false;
  bool same = a->data == b->data && a->ndim == b->ndim;
  for (int i = 0; same && i < a->ndim; i++)
    same = a->shape[i] == b->shape[i] && (a->shape[i] == 1 || a->strides[i] == b->strides[i]);
  if (same) return false;
  // Views into the same rows, side by side (parts of a fused projection's
  // output): equal token strides, disjoint stretches of each row.
  if (a->ndim == 3 && b->ndim == 3 && a->shape[0] == b->shape[0] && a->strides[0] == b->strides[0]) {
    const int64_t row = a->strides[0], d = ((const float*)b->data) - ((const float*)a->data);
    const int64_t la = (a->shape[1] - 1) * a->strides[1] + a->shape[2];
    const int64_t lb = (b->shape[1] - 1) * b->strides[1] + b->shape[2];
    if (d >= la && d + lb <= row) return false;
    if (-d >= lb && -d + la <= row) return false;
  }
  return true;
}

// ---- kernel --------------------------------------------------------------------

struct RotaryDesc {
  const float *q, *k, *v;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  float *qo, *ko;
  int64_t qo_t, qo_h, ko_t, ko_h;
  const float *q_scale, *k_scale, *inv_freq;
  const int* positions;
  float eps, inv_dim;
  int dim, rot, hq, hk, rows;  // rows per token: q, k and, appending, v heads
  CacheView c;
  SeqView s;
};

// The sequence of token t: the last s with q_starts[s] <= t, -1 for none (a
// padding row).  The 64 lanes probe 64 evenly spaced starts at once, so up to
// 64 sequences take one round trip to memory, up to 4096 two.
__device__ __forceinline__ int find_seq(const SeqView& v, int t) {
  if (!v.q_starts) return t;
  const int lane = threadIdx.x & 63;
  int lo = 0, len = v.n + 1;
  while (true) {
    const int step = (len + 63) >> 6;
    const int at = lo + lane * step;
    const bool below = lane * step < len && v.q_starts[at] <= t;
    const int n = __popcll(__ballot(below));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    if (step == 1) return lo < v.n ? lo : -1;
    len = min(step, v.n + 1 - lo);
  }
}

// cos and sin of pos * f, rounded once.  The angle is formed and brought within
// a quarter of pi in 64 bits (at position 10^6 its error is 10^-10; in 32 bits
// it would be 0.06), and so are the Taylor series of sin and cos: the first
// terms left out, x^13 / 13! and x^14 / 14!, are below 2^-36 there.
__device__ __forceinline__ void turn_of(double pos, float f, float& c, float& s) {
  const double angle = pos * (double)f;
  const double n = __builtin_rint(angle * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, angle);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
  const double x2 = r * r;
  double ps = __builtin_fma(x2, -1. / 39916800., 1. / 362880.);
  ps = __builtin_fma(x2, ps, -1. / 5040.);
  ps = __builtin_fma(x2, ps, 1. / 120.);
  ps = __builtin_fma(x2, ps, -1. / 6.);
  const float sn = (float)__builtin_fma(r * x2, ps, r);
  double pc = __builtin_fma(x2, 1. / 479001600., -1. / 3628800.);
  pc = __builtin_fma(x2, pc, 1. / 40320.);
  pc = __builtin_fma(x2, pc, -1. / 720.);
  pc = __builtin_fma(x2, pc, 1. / 24.);
  pc = __builtin_fma(x2, pc, -1. / 2.);
  const float cs = (float)__builtin_fma(x2, pc, 1.);
  const int q = (int)(long long)n & 3;
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  c = (q == 1 || q == 2) ? -a : a;
  s = q >= 2 ? -b : b;
}

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));

// One float4 into a cache row of type TYPE (rtenhip_cache_dtype).
template <int TYPE>
__device__ __forceinline__ void store4(char* row, int at, const float* x) {
  if constexpr (TYPE == RTENHIP_CACHE_F32) {
    *(float4*)(row + (int64_t)at * 4) = make_float4(x[0], x[1], x[2], x[3]);
  } else if constexpr (TYPE == RTENHIP_CACHE_F16) {
    const half4 y = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    *(half4*)(row + (int64_t)at * 2) = y;
  } else {
    const bf4 y = {(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
    *(bf4*)(row + (int64_t)at * 2) = y;
  }
}

constexpr int ROT_THREADS = 256;
constexpr int ROT_AHEAD = 4;  // rows a lane has in flight

// One token per workgroup (blockIdx.x); LPR lanes per head row, each with the
// 8 elements of four pairs, so a row needs no exchange but the sum of its
// squares.  The token's turns are formed once, one by a thread, and shared
// through LDS (8192 tokens of 4 + 2 heads of 128 take 15.3 us, and 17.5 where
// each lane forms its four, in 32 bits).
// gridDim.y workgroups share a token's rows where there are few tokens.
// Bound by memory: rows are read once and written once.  8192 tokens of 32 + 8
// heads of 128 into a bf16 cache, 369 MB: 71.5 us, 5.2 TB/s (a copy of 4 GiB:
// 4.7); one token 3.2 us, a launch.
template <int LPR, int TYPE, bool APPEND, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotaryDesc d) {
  constexpr int RPP = ROT_THREADS / LPR;  // rows per pass of the workgroup
  __shared__ __attribute__((aligned(16))) float cos_sh[ROT_THREADS / 2], sin_sh[ROT_THREADS / 2];
  const int t = blockIdx.x;
  const int j = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  const bool live = j * 8 < d.dim, turned = j * 8 < d.rot;
  // The lane's two groups of four elements.
  const int o0 = !INTER && turned ? 4 * j : 8 * j;
  const int o1 = !INTER && turned ? d.rot / 2 + 4 * j : 8 * j + 4;

  int pos = 0, page = -1, slot = 0;
  if (APPEND) {
    const int s = find_seq(d.s, t);
    if (s < 0) return;  // padding
    const int end = d.s.q_starts ? d.s.q_starts[s + 1] : t + 1;
    pos = d.s.kv_lens[s] - (end - t);
    if (pos >= 0) {
      page = page_entry(d.s.table + (int64_t)s * d.s.table_stride, d.s.max_pages, d.c, pos);
      slot = pos - fdiv(pos, d.c.page_div) * d.c.page_size;
    }
  }
  if (d.positions) pos = d.positions[t];
  float4 cs4 = make_float4(1.f, 1.f, 1.f, 1.f), sn4 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d.rot) {
    if ((int)threadIdx.x < d.rot / 2) {
      float c, s;
      turn_of((double)pos, d.inv_freq[threadIdx.x], c, s);
      cos_sh[threadIdx.x] = c, sin_sh[threadIdx.x] = s;
    }
    __syncthreads();  // (padding has left as a whole)
    if (turned) cs4 = *(const float4*)&cos_sh[4 * j], sn4 = *(const float4*)&sin_sh[4 * j];
  }
  const float cs[4] = {cs4.x, cs4.y, cs4.z, cs4.w}, sn[4] = {sn4.x, sn4.y, sn4.z, sn4.w};

  for (int r0 = (blockIdx.y * RPP) + sub; r0 < d.rows; r0 += gridDim.y * RPP * ROT_AHEAD) {
    float x[ROT_AHEAD][8];
#pragma unroll
    for (int u = 0; u < ROT_AHEAD; u++) {
      const int r = r0 + u * gridDim.y * RPP;
      if (r < d.rows && live) {
        const float* p;
        if (r < d.hq) p = d.q + t * d.q_t + r * d.q_h;
        else if (!APPEND || r < d.hq + d.hk) p = d.k + t * d.k_t + (r - d.hq) * d.k_h;
        else p = d.v + t * d.v_t + (r - d.hq - d.hk) * d.v_h;
        const float4 a = *(const float4*)(p + o0), b = *(const float4*)(p + o1);
        x[u][0] = a.x, x[u][1] = a.y, x[u][2] = a.z, x[u][3] = a.w;
        x[u][4] = b.x, x[u][5] = b.y, x[u][6] = b.z, x[u][7] = b.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[u][e] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < ROT_AHEAD; u++) {
      const int r = r0 + u * gridDim.y * RPP;
      if (r >= d.rows) continue;
      const bool is_v = APPEND && r >= d.hq + d.hk;
      float* y = x[u];
      if (!is_v) {
        const float* w = r < d.hq ? d.q_scale : d.k_scale;
        if (w) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; e++) ss = __fmaf_rn(y[e], y[e], ss);
#pragma unroll
          for (int m = LPR / 2; m; m >>= 1) ss += __shfl_xor(ss, m, LPR);
          const float inv = 1.f / sqrtf(__fmaf_rn(ss, d.inv_dim, d.eps));
          if (live) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              y[e] = y[e] * inv * w[o0 + e];
              y[4 + e] = y[4 + e] * inv * w[o1 + e];
            }
          }
        }
        if (turned) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : i + 4;
            const float a = y[ia], b = y[ib];
            y[ia] = __fmaf_rn(a, cs[i], -(b * sn[i]));
            y[ib] = __fmaf_rn(b, cs[i], a * sn[i]);
          }
        }
      }
      if (!live) continue;
      if (r < d.hq || !APPEND) {
        float* p = r < d.hq ? d.qo + t * d.qo_t + r * d.qo_h : d.ko + t * d.ko_t + (r - d.hq) * d.ko_h;
        *(float4*)(p + o0) = make_float4(y[0], y[1], y[2], y[3]);
        *(float4*)(p + o1) = make_float4(y[4], y[5], y[6], y[7]);
      } else if (page_ok(d.c, page)) {
        constexpr int size = TYPE == RTENHIP_CACHE_F32 ? 4 : 2;
        char* row = is_v ? d.c.v + (page * d.c.v_page + slot * d.c.v_slot + (r - d.hq - d.hk) * d.c.v_head) * size
                         : d.c.k + (page * d.c.k_page + slot * d.c.k_slot + (r - d.hq) * d.c.k_head) * size;
        store4<TYPE>(row, o0, y);
        store4<TYPE>(row, o1, y + 4);
      }
    }
  }
}

template <int TYPE, bool APPEND, bool INTER>
static rtenhip_status launch_rotary(const RotaryDesc& d, int64_t tokens, hipStream_t s) {
  const int lpr = d.dim <= 64 ? 8 : d.dim <= 128 ? 16 : 32;
  const int rpp = ROT_THREADS / lpr;
  // Few tokens: a workgroup per pass of a token's rows, so that no load waits
  // for another; many tokens fill the card by themselves and then share the
  // turns among all rows.  (32 + 8 heads of 128: one token 3.2 against 4.4 us
  // with one workgroup, 400 tokens 5.9 and 6.2, 1024 10.3 and 10.1, 8192 74 and
  // 71.5.)
  const int passes = (d.rows + rpp - 1) / rpp;
  const dim3 grid((unsigned)tokens, (unsigned)(tokens < 512 ? passes : 1));
  if (lpr == 8)
    hipLaunchKernelGGL((rotary_kernel<8, TYPE, APPEND, INTER>), grid, dim3(ROT_THREADS), 0, s, d);
  else if (lpr == 16)
    hipLaunchKernelGGL((rotary_kernel<16, TYPE, APPEND, INTER>), grid, dim3(ROT_THREADS), 0, s, d);
  else
    hipLaunchKernelGGL((rotary_kernel<32, TYPE, APPEND, INTER>), grid, dim3(ROT_THREADS), 0, s, d);
  RTENHIP_LAUNCH_CHECK();
  return RTENHIP_OK;
}

// The checks and the descriptor parts both entry points have in common.
static rtenhip_status rotary_desc(const rtenhip_tensor* q, const rtenhip_tensor* k, const rtenhip_rotary* r,
                                  const rtenhip_tensor* q_out, RotaryDesc& d) {
  if (!q || !k || !r || !q_out) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  if (q->ndim != 3 || k->ndim != 3)
    return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Expected [tokens, heads, head_dim] inputs");
  const int64_t tokens = q->shape[0], dim = q->shape[2];
  if (dim < 8 || dim > 256 || dim % 8)
    return fail(RTENHIP_UNSUPPORTED_VALUE, "head_dim must be a multiple of 8 from 8 to 256");
  if (tokens < 0 || tokens > INT32_MAX || q->shape[1] < 0 || q->shape[1] > 65536 || k->shape[1] < 0 ||
      k->shape[1] > 65536)
    return fail(RTENHIP_INVALID_VALUE, "Invalid input size");
  if (!launchable(tokens, ROT_THREADS)) return fail(RTENHIP_UNSUPPORTED_VALUE, "Too many tokens");
  if (r->rotary_dim < 0 || r->rotary_dim > dim || r->rotary_dim % 8)
    return fail(RTENHIP_UNSUPPORTED_VALUE, "rotary_dim must be a multiple of 8 up to head_dim");
  if (!(r->epsilon >= 0.f)) return fail(RTENHIP_INVALID_VALUE, "epsilon must not be negative");
  if (r->rotary_dim && !r->inv_freq) return fail(RTENHIP_MISSING_INPUTS, "Missing inv_freq");
  for (const void* p : {(const void*)r->q_scale, (const void*)r->k_scale, (const void*)r->inv_freq,
                        (const void*)r->positions})
    if ((uintptr_t)p % 4) return fail(RTENHIP_UNSUPPORTED_VALUE, "Scales, frequencies and positions must be on 4 bytes");
  const char* shape = "q, k and their outputs must be [tokens, heads, head_dim] of the same tokens and head_dim";
  const char* align = "Head rows must have unit stride and start on 16 bytes";
  rtenhip_status st = check_rows(q, tokens, q->shape[1], dim, shape, align);
  if (!st) st = check_rows(k, tokens, k->shape[1], dim, shape, align);
  if (!st) st = check_rows(q_out, tokens, q->shape[1], dim, shape, align);
  if (st) return st;
  if (!rows_apart(q_out->shape, q_out->strides, 2, dim))
    return fail(RTENHIP_INVALID_VALUE, "Output rows must not overlap");
  d.q = q->data, d.q_t = q->strides[0], d.q_h = q->strides[1];
  d.k = k->data, d.k_t = k->strides[0], d.k_h = k->strides[1];
  d.qo = q_out->data, d.qo_t = q_out->strides[0], d.qo_h = q_out->strides[1];
  d.q_scale = r->q_scale, d.k_scale = r->k_scale, d.inv_freq = r->inv_freq, d.positions = r->positions;
  d.eps = r->epsilon;
  d.inv_dim = 1.f / (float)dim;
  d.dim = (int)dim, d.rot = r->rotary_dim, d.hq = (int)q->shape[1], d.hk = (int)k->shape[1];
  return RTENHIP_OK;
}

}  // namespace rtenhip

using namespace rtenhip;

extern "C" rtenhip_status rtenhip_qk_norm_rotary_f32(rtenhip_ctx* ctx, const rtenhip_tensor* q,
                                                     const rtenhip_tensor* k, const rtenhip_rotary* r,
                                                     rtenhip_tensor* q_out, rtenhip_tensor* k_out) {
  RotaryDesc d{};
  rtenhip_status st = rotary_desc(q, k, r, q_out, d);
  if (!st)
    st = check_rows(k_out, q->shape[0], k->shape[1], q->shape[2],
                    "q, k and their outputs must be [tokens, heads, head_dim] of the same tokens and head_dim",
                    "Head rows must have unit stride and start on 16 bytes");
  if (st) return st;
  if (!r->positions && r->rotary_dim && q->shape[0]) return fail(RTENHIP_MISSING_INPUTS, "Missing positions");
  if (!rows_apart(k_out->shape, k_out->strides, 2, q->shape[2]))
    return fail(RTENHIP_INVALID_VALUE, "Output rows must not overlap");
  if (rows_clash(q, q_out) || rows_clash(k, k_out) || rows_clash(q_out, k_out) || rows_clash(q, k_out) ||
      rows_clash(k, q_out) || (q_out->data == k_out->data && numel(*q_out) && numel(*k_out)) ||
      (q->data == k_out->data && numel(*q) && numel(*k)) || (k->data == q_out->data && numel(*q) && numel(*k)))
    return fail(RTENHIP_INVALID_VALUE, "Outputs may share memory with their own input only");
  if (!ctx) return fail(RTENHIP_MISSING_INPUTS, "Missing context");
  d.ko = k_out->data, d.ko_t = k_out->strides[0], d.ko_h = k_out->strides[1];
  d.rows = d.hq + d.hk;
  if (q->shape[0] == 0 || d.rows == 0) return RTENHIP_OK;
  DeviceScope on(reinterpret_cast<Ctx*>(ctx)->device);
  if (on.status) return on.status;
  return r->interleaved ? launch_rotary<RTENHIP_CACHE_F32, false, true>(d, q->shape[0], stream_of(ctx))
                        : launch_rotary<RTENHIP_CACHE_F32, false, false>(d, q->shape[0], stream_of(ctx));
}

extern "C" rtenhip_status rtenhip_qk_norm_rotary_append_f32(rtenhip_ctx* ctx, const rtenhip_tensor* q,
                                                            const rtenhip_tensor* k, const rtenhip_tensor* v,
                                                            const rtenhip_rotary* r, const rtenhip_kv_cache* cache,
                                                            const rtenhip_sequences* seqs, rtenhip_tensor* q_out) {
  RotaryDesc d{};
  int dtype = 0;
  rtenhip_status st = rotary_desc(q, k, r, q_out, d);
  if (!st)
    st = check_rows(v, q->shape[0], k->shape[1], q->shape[2], "v must have the shape of k",
                    "Head rows must have unit stride and start on 16 bytes");
  if (!st) st = cache_view(cache, d.c, dtype);
  if (!st) st = seq_view(seqs, q->shape[0], d.s);
  if (st) return st;
  if (d.c.heads != d.hk || d.c.dim != d.dim)
    return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Cache heads and head_dim must be those of k");
  const int64_t extent[3] = {cache->n_pages, cache->page_size, cache->n_heads};
  if (!rows_apart(extent, cache->k_strides, 3, d.dim) || !rows_apart(extent, cache->v_strides, 3, d.dim))
    return fail(RTENHIP_INVALID_VALUE, "Cache rows must not overlap");
  if (rows_clash(q, q_out) || rows_clash(k, q_out) || rows_clash(v, q_out) ||
      (numel(*q) && numel(*k) && (k->data == q_out->data || v->data == q_out->data)))
    return fail(RTENHIP_INVALID_VALUE, "Outputs may share memory with their own input only");
  if (!ctx) return fail(RTENHIP_MISSING_INPUTS, "Missing context");
  d.v = v->data, d.v_t = v->strides[0], d.v_h = v->strides[1];
  d.rows = d.hq + 2 * d.hk;
  if (q->shape[0] == 0 || seqs->n_seqs == 0) return RTENHIP_OK;
  DeviceScope on(reinterpret_cast<Ctx*>(ctx)->device);
  if (on.status) return on.status;
  const int64_t n = q->shape[0];
  hipStream_t s = stream_of(ctx);
  const bool inter = r->interleaved != 0;
  if (dtype == RTENHIP_CACHE_F32)
    return inter ? launch_rotary<RTENHIP_CACHE_F32, true, true>(d, n, s) : launch_rotary<RTENHIP_CACHE_F32, true, false>(d, n, s);
  if (dtype == RTENHIP_CACHE_F16)
    return inter ? launch_rotary<RTENHIP_CACHE_F16, true, true>(d, n, s) : launch_rotary<RTENHIP_CACHE_F16, true, false>(d, n, s);
  return inter ? launch_rotary<RTENHIP_CACHE_BF16, true, true>(d, n, s) : launch_rotary<RTENHIP_CACHE_BF16, true, false>(d, n, s);
}
