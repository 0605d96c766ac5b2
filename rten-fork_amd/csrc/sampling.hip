// One token for each row of logits: temperature, top-k, top-p, min-p and a
// draw from a given random number (rtenhip_sample_f32).
//
// The token is a whole number that has to be the right one, so the weights
// m_i = exp((l_i - max) / T) are formed in 64 bits and summed as integers,
// m_i 2^S rounded, S such that a row's sum stays below 2^63 (S = 45 at 131,072
// tokens): the sums do not depend on any order, and what a weight loses, 2^-46
// of the largest, moves a draw's borders by less than 2^-28.
//
// All filters keep a prefix of the order (falling logit, rising index), which
// needs no sort: a prefix is a key (the logit's bits in their order) above
// which all are kept, and a number of first ones equal to it.  The key is
// found digit by digit (11, 11 and 10 bits) from histograms of counts and
// weights, first the one of top-k, whose weight is what top-p is a share of,
// then that of top-p.  The draw then needs the kept weight of each block of
// 2048 tokens and one look into the block that it falls into.
//
// One launch per pass over the logits, the rows cut into enough stretches to
// fill the card; every workgroup repeats the small decision that the pass
// before has made possible.  Passes nobody asks for are left out: without a
// filter three remain.
#include "decoder.h"

#include <algorithm>
#include <cmath>

namespace rtenhip {

typedef unsigned long long u64;

constexpr int SA_THREADS = 256;
constexpr int SA_BLOCK = 2048;  // tokens of a sum
constexpr int SA_BINS = 2048;
constexpr float SA_NEG_INF = -__builtin_huge_valf();

struct Bin {
  u64 mass;
  u64 count;
};

// What is known of a row so far.
struct RowState {
  u64 total;       // weight of all tokens, then of the top-k set
  u64 k_above, p_above;  // weight above the digit / key found so far
  u64 n_above;     // tokens above it (top-k)
  uint32_t k_key, p_key;
  int k_on, p_on;  // a limit was found
  u64 ties;        // of the final key
  uint32_t key;    // final: kept are keys above it, and the first `ties` equal to it
};

struct SampleDesc {
  const float* logits;
  int64_t row_stride;
  int rows, vocab, cuts, per_cut, blocks;  // blocks of SA_BLOCK; per_cut of them to a workgroup
  int shift;
  rtenhip_sampling f;
  const float* uniforms;
  int* tokens;
  float* logprobs;
  // Workspace.
  float* cut_max;   // [rows][cuts]
  int* cut_arg;     // [rows][cuts]
  // [rows], one for each pass that decides something: a pass reads the last
  // one's (null: nothing is known yet) while its first workgroups write its own.
  RowState* states[5];
  const RowState* from;
  RowState* to;
  u64* block_mass;  // [rows][blocks]
  int* block_ties;  // [rows][blocks]
  Bin* hist[5];     // [rows][SA_BINS]: first digit; top-k's second, third; top-p's
};

struct Filters {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy;
};

__device__ __forceinline__ Filters filters_of(const SampleDesc& d, int row) {
  Filters f;
  f.temperature = d.f.temperatures ? d.f.temperatures[row] : d.f.temperature;
  f.top_p = d.f.top_ps ? d.f.top_ps[row] : d.f.top_p;
  f.min_p = d.f.min_ps ? d.f.min_ps[row] : d.f.min_p;
  f.top_k = d.f.top_ks ? d.f.top_ks[row] : d.f.top_k;
  f.greedy = !(f.temperature > 0.f);
  return f;
}

// Falling logits are falling keys; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// exp(x) for x <= 0 to 2^-50: 2^n times the Taylor series of exp(r),
// |r| <= ln 2 / 2, whose first term left out is r^13 / 13! < 2^-52.
__device__ __forceinline__ double exp_nonpos(double x) {
  x = x < -700. ? -700. : x;
  const double n = __builtin_rint(x * 1.44269504088896340736);
  double r = __builtin_fma(n, -6.93147180369123816490e-01, x);
  r = __builtin_fma(n, -1.90821492927058770002e-10, r);
  double p = 1. / 479001600.;
  p = __builtin_fma(p, r, 1. / 39916800.);
  p = __builtin_fma(p, r, 1. / 3628800.);
  p = __builtin_fma(p, r, 1. / 362880.);
  p = __builtin_fma(p, r, 1. / 40320.);
  p = __builtin_fma(p, r, 1. / 5040.);
  p = __builtin_fma(p, r, 1. / 720.);
  p = __builtin_fma(p, r, 1. / 120.);
  p = __builtin_fma(p, r, 1. / 24.);
  p = __builtin_fma(p, r, 1. / 6.);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.);
  p = __builtin_fma(p, r, 1.);
  return ldexp(p, (int)n);
}

// A row's weights.
struct Weigh {
  double max, inv_t, up, min_p;
  bool infinite;
  __device__ Weigh(const SampleDesc& d, const Filters& f, float row_max) {
    max = row_max;
    inv_t = 1. / (double)f.temperature;
    up = ldexp(1., d.shift);
    min_p = f.min_p > 1.f ? 1. : f.min_p > 0.f ? (double)f.min_p : 0.;
    infinite = row_max == -SA_NEG_INF;
  }
  // m 2^S as an integer (S <= 51: the sum with 2^52 holds it in its low
  // bits); 0 for what can not be taken.
  __device__ __forceinline__ u64 operator()(float x, bool min_filter) const {
    if (infinite) return x == -SA_NEG_INF ? (u64)up : 0;
    if (!(x > SA_NEG_INF)) return 0;
    const double e = exp_nonpos(((double)x - max) * inv_t);
    if (min_filter && e < min_p) return 0;
    return (u64)__double_as_longlong(__builtin_fma(e, up, 4503599627370496.)) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ u64 wave_scan64(u64 x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const u64 y = __shfl_up((unsigned long long)x, m);
    if (lane >= m) x += y;
  }
  return x;
}

// Exclusive prefix over the workgroup's 256 threads; `all` is the sum.
__device__ __forceinline__ u64 block_scan(u64 x, u64* sh, u64& all) {
  const u64 in = wave_scan64(x);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[wave] = in;
  __syncthreads();
  u64 at = in - x;
  all = 0;
#pragma unroll
  for (int w = 0; w < SA_THREADS / 64; w++) {
    if (w < wave) at += sh[w];
    all += sh[w];
  }
  return at;
}

// The largest logit of a row from the stretches' ones.
__device__ __forceinline__ float row_max_of(const SampleDesc& d, int row, float* sh) {
  float m = SA_NEG_INF;
  for (int i = threadIdx.x; i < d.cuts; i += SA_THREADS) m = fmaxf(m, d.cut_max[(int64_t)row * d.cuts + i]);
#pragma unroll
  for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

// The bin, from the highest down, at which the counts (or weights) reach
// `target`: found, with the sums above it.  The whole workgroup calls it.
struct Found {
  int bin;  // -1: the sum of all is less than target
  u64 count_above, mass_above, count_all, mass_all;
};
__device__ Found find_bin(const Bin* hist, bool by_mass, u64 target, u64* sh, Found* found) {
  constexpr int EACH = SA_BINS / SA_THREADS;
  const int top = SA_BINS - 1 - threadIdx.x * EACH;
  u64 count = 0, mass = 0;
  Bin b[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    b[i] = hist[top - i];
    count += b[i].count;
    mass += b[i].mass;
  }
  Found r;
  u64 c = block_scan(count, sh, r.count_all), m = block_scan(mass, sh, r.mass_all);
  if (threadIdx.x == 0) found->bin = -1;
  __syncthreads();
  if ((by_mass ? m : c) < target && (by_mass ? m + mass : c + count) >= target) {
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if ((by_mass ? m : c) < target && (by_mass ? m + b[i].mass : c + b[i].count) >= target) {
        found->bin = top - i;
        found->count_above = c;
        found->mass_above = m;
      }
      c += b[i].count;
      m += b[i].mass;
    }
  }
  __syncthreads();
  r.bin = found->bin;
  r.count_above = found->count_above;
  r.mass_above = found->mass_above;
  __syncthreads();
  return r;
}

// ceil(share of the kept weight), at least 1 so that the first token stays.
__device__ __forceinline__ u64 p_target(float p, u64 total) {
  const double t = __builtin_ceil((p > 0.f ? (double)p : 0.) * (double)total);
  const u64 n = (u64)t;
  return n < 1 ? 1 : n > total ? total : n;
}

enum SamplePass { PASS_FIRST, PASS_K2, PASS_K3, PASS_P2, PASS_P3, PASS_SUM };

struct SampleShared {
  u64 scan[SA_THREADS / 64];
  float top[SA_THREADS / 64];
  Found found;
};

// What the histograms so far say of a row, given what had been known before:
// every workgroup of the row comes to the same.
__device__ void decide(const SampleDesc& d, int pass, int row, const Filters& f, const Weigh& weigh, RowState& st,
                       SampleShared& sh) {
  const int64_t at = (int64_t)row * SA_BINS;
  const bool k_asked = f.top_k > 0, p_asked = f.top_p < 1.f;
  st = d.from ? d.from[row] : RowState{};
  if (pass == PASS_K2) {
    const Found r = find_bin(d.hist[0] + at, false, k_asked ? (u64)f.top_k : ~0ull, sh.scan, &sh.found);
    st.total = r.mass_all;
    st.k_on = k_asked && r.bin >= 0;
    st.k_key = (uint32_t)r.bin << 21;
    st.k_above = r.mass_above;
    st.n_above = r.count_above;
  } else if (pass == PASS_K3) {
    if (!st.k_on) return;
    const Found r = find_bin(d.hist[1] + at, false, (u64)f.top_k - st.n_above, sh.scan, &sh.found);
    st.k_key |= (uint32_t)r.bin << 10;
    st.k_above += r.mass_above;
    st.n_above += r.count_above;
  } else if (pass == PASS_P2) {
    if (st.k_on) {
      const Found r = find_bin(d.hist[2] + at, false, (u64)f.top_k - st.n_above, sh.scan, &sh.found);
      st.k_key |= (uint32_t)r.bin;
      st.k_above += r.mass_above;
      st.n_above += r.count_above;
      st.ties = (u64)f.top_k - st.n_above;
      st.key = st.k_key;
      st.total = st.k_above + st.ties * weigh(of_key(st.k_key), false);
    }
    if (p_asked) {
      Found r = find_bin(d.hist[0] + at, true, ~0ull, sh.scan, &sh.found);
      if (!st.k_on) st.total = r.mass_all;
      r = find_bin(d.hist[0] + at, true, p_target(f.top_p, st.total), sh.scan, &sh.found);
      st.p_on = r.bin >= 0;
      st.p_key = (uint32_t)r.bin << 21;
      st.p_above = r.mass_above;
    }
  } else if (pass == PASS_P3) {
    if (!st.p_on) return;
    const Found r = find_bin(d.hist[3] + at, true, p_target(f.top_p, st.total) - st.p_above, sh.scan, &sh.found);
    st.p_key |= (uint32_t)r.bin << 10;
    st.p_above += r.mass_above;
  } else if (pass == PASS_SUM) {
    if (d.hist[3]) {
      if (st.p_on) {
        const u64 target = p_target(f.top_p, st.total);
        const Found r = find_bin(d.hist[4] + at, true, target - st.p_above, sh.scan, &sh.found);
        st.key = st.p_key | (uint32_t)r.bin;
        const u64 one = weigh(of_key(st.key), false), left = target - st.p_above - r.mass_above;
        st.ties = one ? (left + one - 1) / one : 0;
      } else if (!st.k_on) {
        st.key = 0, st.ties = 0;
      }
    } else if (st.k_on) {
      const Found r = find_bin(d.hist[2] + at, false, (u64)f.top_k - st.n_above, sh.scan, &sh.found);
      st.key = st.k_key | (uint32_t)r.bin;
      st.ties = (u64)f.top_k - st.n_above - r.count_above;
    } else {
      st.key = 0, st.ties = 0;
    }
  }
}

// Largest logit, and its first place, of each stretch; clears the histograms.
__global__ __launch_bounds__(SA_THREADS) void sample_top_kernel(SampleDesc d) {
  __shared__ float m_sh[SA_THREADS / 64];
  __shared__ int i_sh[SA_THREADS / 64];
  const int row = blockIdx.x / d.cuts, cut = blockIdx.x - row * d.cuts;
  const int i0 = cut * d.per_cut * SA_BLOCK, i1 = min(d.vocab, i0 + d.per_cut * SA_BLOCK);
  const float* x = d.logits + (int64_t)row * d.row_stride;
  float m = SA_NEG_INF;
  int arg = 0x7fffffff;
#pragma unroll 8
  for (int i = i0 + threadIdx.x; i < i1; i += SA_THREADS) {
    const float v = x[i];
    if (v > m) m = v, arg = i;  // (never for a NaN)
  }
  for (int h = 0; h < 5; h++)
    if (d.hist[h])
      for (int i = cut * SA_THREADS + threadIdx.x; i < SA_BINS; i += d.cuts * SA_THREADS)
        d.hist[h][(int64_t)row * SA_BINS + i] = Bin{0, 0};
#pragma unroll
  for (int k = 32; k; k >>= 1) {
    const float m2 = __shfl_xor(m, k);
    const int a2 = __shfl_xor(arg, k);
    if (m2 > m || (m2 == m && a2 < arg)) m = m2, arg = a2;
  }
  if ((threadIdx.x & 63) == 0) m_sh[threadIdx.x >> 6] = m, i_sh[threadIdx.x >> 6] = arg;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < SA_THREADS / 64; w++)
      if (m_sh[w] > m || (m_sh[w] == m && i_sh[w] < arg)) m = m_sh[w], arg = i_sh[w];
    d.cut_max[(int64_t)row * d.cuts + cut] = m;
    d.cut_arg[(int64_t)row * d.cuts + cut] = arg;
  }
}

// One digit's histogram of a row's stretch: PASS_FIRST of all tokens, the
// others of those whose digits so far are those found.
template <int PASS>
__global__ __launch_bounds__(SA_THREADS) void sample_hist_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ u64 mass_sh[SA_BINS];
  __shared__ uint32_t count_sh[SA_BINS];
  const int row = blockIdx.x / d.cuts, cut = blockIdx.x - row * d.cuts;
  const Filters f = filters_of(d, row);
  const float top = row_max_of(d, row, sh.top);
  if (f.greedy || top == SA_NEG_INF) return;
  const Weigh weigh(d, f, top);
  uint32_t prefix = 0;
  if (PASS != PASS_FIRST) {
    RowState st;
    decide(d, PASS, row, f, weigh, st, sh);
    __syncthreads();
    if (cut == 0 && threadIdx.x == 0) d.to[row] = st;
    if (PASS == PASS_K2 || PASS == PASS_K3 ? !st.k_on : !st.p_on) return;
    prefix = PASS == PASS_K2 || PASS == PASS_K3 ? st.k_key : st.p_key;
  }
  for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) mass_sh[i] = 0, count_sh[i] = 0;
  __syncthreads();
  const int i0 = cut * d.per_cut * SA_BLOCK, i1 = min(d.vocab, i0 + d.per_cut * SA_BLOCK);
  const float* x = d.logits + (int64_t)row * d.row_stride;
#pragma unroll 4
  for (int i = i0 + threadIdx.x; i < i1; i += SA_THREADS) {
    const float v = x[i];
    const uint32_t key = key_of(v);
    if (PASS == PASS_K2 || PASS == PASS_P2)
      if (key >> 21 != prefix >> 21) continue;
    if (PASS == PASS_K3 || PASS == PASS_P3)
      if (key >> 10 != prefix >> 10) continue;
    const u64 m = weigh(v, false);
    if (!m) continue;
    const int bin = PASS == PASS_FIRST ? key >> 21 : PASS == PASS_K2 || PASS == PASS_P2 ? key >> 10 & 2047 : key & 1023;
    atomicAdd(&mass_sh[bin], m);
    atomicAdd(&count_sh[bin], 1u);
  }
  __syncthreads();
  Bin* to = d.hist[PASS] + (int64_t)row * SA_BINS;
  for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS)
    if (count_sh[i]) {
      atomicAdd(&to[i].mass, mass_sh[i]);
      atomicAdd(&to[i].count, (u64)count_sh[i]);
    }
}

// Kept weight above the key, and the number of ties, of each block.
__global__ __launch_bounds__(SA_THREADS) void sample_sum_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ u64 m_sh[SA_THREADS / 64];
  __shared__ int t_sh[SA_THREADS / 64];
  const int row = blockIdx.x / d.cuts, cut = blockIdx.x - row * d.cuts;
  const Filters f = filters_of(d, row);
  const float top = row_max_of(d, row, sh.top);
  if (f.greedy || top == SA_NEG_INF) return;
  const Weigh weigh(d, f, top);
  RowState st;
  decide(d, PASS_SUM, row, f, weigh, st, sh);
  __syncthreads();
  if (cut == 0 && threadIdx.x == 0) d.to[row] = st;
  const float* x = d.logits + (int64_t)row * d.row_stride;
  const int b1 = min(d.blocks, (cut + 1) * d.per_cut);
  for (int b = cut * d.per_cut; b < b1; b++) {
    u64 mass = 0;
    int ties = 0;
#pragma unroll
    for (int u = 0; u < SA_BLOCK / SA_THREADS; u++) {
      const int i = b * SA_BLOCK + u * SA_THREADS + threadIdx.x;
      const float v = i < d.vocab ? x[i] : SA_NEG_INF;
      const uint32_t key = key_of(v);
      if (key > st.key) mass += weigh(v, true);
      ties += st.ties && key == st.key && weigh(v, true);
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) mass += __shfl_xor((unsigned long long)mass, k), ties += __shfl_xor(ties, k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) m_sh[threadIdx.x >> 6] = mass, t_sh[threadIdx.x >> 6] = ties;
    __syncthreads();
    if (threadIdx.x == 0) {
      d.block_mass[(int64_t)row * d.blocks + b] = m_sh[0] + m_sh[1] + m_sh[2] + m_sh[3];
      d.block_ties[(int64_t)row * d.blocks + b] = t_sh[0] + t_sh[1] + t_sh[2] + t_sh[3];
    }
  }
}

// The draw: the block, then the token.
__global__ __launch_bounds__(SA_THREADS) void sample_pick_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ u64 base_sh, ties_sh;
  __shared__ int block_sh;
  const int row = blockIdx.x, tid = threadIdx.x;
  const Filters f = filters_of(d, row);
  const float top = row_max_of(d, row, sh.top);
  if (f.greedy || top == SA_NEG_INF) {
    if (tid == 0) {
      int arg = 0x7fffffff;
      for (int i = 0; i < d.cuts; i++)
        if (d.cut_max[(int64_t)row * d.cuts + i] == top) arg = min(arg, d.cut_arg[(int64_t)row * d.cuts + i]);
      d.tokens[row] = top == SA_NEG_INF ? -1 : arg;
      if (d.logprobs) d.logprobs[row] = top == SA_NEG_INF ? SA_NEG_INF : 0.f;
    }
    return;
  }
  const Weigh weigh(d, f, top);
  const RowState st = d.from[row];
  const u64 one = st.ties ? weigh(of_key(st.key), true) : 0;
  // Blocks, a stretch of them to each thread.
  const int each = (d.blocks + SA_THREADS - 1) / SA_THREADS;
  const int b0 = min(d.blocks, tid * each), b1 = min(d.blocks, b0 + each);
  const u64* bm = d.block_mass + (int64_t)row * d.blocks;
  const int* bt = d.block_ties + (int64_t)row * d.blocks;
  u64 ties = 0, all;
  for (int b = b0; b < b1; b++) ties += bt[b];
  u64 ties_at = block_scan(ties, sh.scan, all);
  const auto kept = [&](u64 before, u64 n) {  // of n ties behind `before` others
    return before >= st.ties ? 0 : min(n, st.ties - before);
  };
  u64 mass = 0, t = ties_at;
  for (int b = b0; b < b1; b++) {
    mass += bm[b] + kept(t, bt[b]) * one;
    t += bt[b];
  }
  u64 total;
  u64 at = block_scan(mass, sh.scan, total);
  float u = d.uniforms[row];
  u = !(u > 0.f) ? 0.f : u >= 1.f ? 0.99999994f : u;
  u64 draw = (u64)((double)u * (double)total);
  draw = min(draw, total - 1);
  if (draw >= at && draw < at + mass) {
    t = ties_at;
    for (int b = b0; b < b1; b++) {
      const u64 m = bm[b] + kept(t, bt[b]) * one;
      if (draw < at + m) {
        block_sh = b, base_sh = at, ties_sh = t;
        break;
      }
      at += m;
      t += bt[b];
    }
  }
  __syncthreads();
  // Tokens, SA_BLOCK / SA_THREADS neighbours to each thread.
  constexpr int EACH = SA_BLOCK / SA_THREADS;
  const float* x = d.logits + (int64_t)row * d.row_stride;
  const int i0 = block_sh * SA_BLOCK + tid * EACH;
  u64 m[EACH];
  bool tie[EACH];
  ties = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const float v = i0 + i < d.vocab ? x[i0 + i] : SA_NEG_INF;
    const uint32_t key = key_of(v);
    m[i] = key >= st.key ? weigh(v, true) : 0;
    tie[i] = key == st.key && m[i];
    ties += tie[i];
  }
  ties_at = ties_sh + block_scan(ties, sh.scan, all);
  mass = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    if (tie[i]) m[i] = ties_at++ < st.ties ? m[i] : 0;
    mass += m[i];
  }
  at = base_sh + block_scan(mass, sh.scan, all);
  if (draw >= at && draw < at + mass) {
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      if (draw >= at && draw < at + m[i]) {
        d.tokens[row] = i0 + i;
        if (d.logprobs) d.logprobs[row] = (float)log((double)m[i] / (double)total);
      }
      at += m[i];
    }
  }
}

// ---- host ----------------------------------------------------------------------------

static int log2_up(int64_t n) {
  int k = 0;
  while ((int64_t(1) << k) < n) k++;
  return k;
}

static rtenhip_status sample_sizes(int64_t rows, int64_t vocab, SampleDesc& d) {
  if (rows < 0 || vocab < 1) return fail(RTENHIP_INVALID_VALUE, "Invalid logits size");
  if (vocab > (int64_t(1) << 24)) return fail(RTENHIP_UNSUPPORTED_VALUE, "Vocabulary is too large");
  if (rows > (int64_t(1) << 20)) return fail(RTENHIP_UNSUPPORTED_VALUE, "Too many rows");
  d.rows = (int)rows;
  d.vocab = (int)vocab;
  d.blocks = (int)((vocab + SA_BLOCK - 1) / SA_BLOCK);
  // Workgroups for the whole card (four to a CU) where the rows alone are
  // too few.
  const int want = rows ? (int)std::max<int64_t>(1, 1024 / rows) : 1;
  d.per_cut = (d.blocks + want - 1) / want;
  d.cuts = (d.blocks + d.per_cut - 1) / d.per_cut;
  d.shift = std::min(51, 62 - log2_up(vocab));
  return RTENHIP_OK;
}

// Lays the workspace out from `base`; its size.  The size does not depend on
// the filters: histograms nobody needs are left alone.
static size_t sample_layout(SampleDesc& d, char* base) {
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* p = base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  d.cut_max = (float*)take((size_t)d.rows * d.cuts * 4);
  d.cut_arg = (int*)take((size_t)d.rows * d.cuts * 4);
  for (int i = 0; i < 5; i++) d.states[i] = (RowState*)take((size_t)d.rows * sizeof(RowState));
  d.block_mass = (u64*)take((size_t)d.rows * d.blocks * 8);
  d.block_ties = (int*)take((size_t)d.rows * d.blocks * 4);
  for (int h = 0; h < 5; h++) d.hist[h] = (Bin*)take((size_t)d.rows * SA_BINS * sizeof(Bin));
  return at;
}

}  // namespace rtenhip

using namespace rtenhip;

extern "C" rtenhip_status rtenhip_sample_workspace(int64_t rows, int64_t vocab, size_t* bytes) {
  if (!bytes) return fail(RTENHIP_MISSING_INPUTS, "Missing output");
  SampleDesc d{};
  const rtenhip_status st = sample_sizes(rows, vocab, d);
  if (st) return st;
  *bytes = sample_layout(d, nullptr);
  return RTENHIP_OK;
}

extern "C" rtenhip_status rtenhip_sample_f32(rtenhip_ctx* ctx, const rtenhip_tensor* logits,
                                             const rtenhip_sampling* sampling, const float* uniforms, void* workspace,
                                             size_t workspace_bytes, int32_t* tokens, float* logprobs) {
  if (!logits || !sampling) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  if (logits->ndim != 2) return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Expected [rows, vocab] logits");
  SampleDesc d{};
  rtenhip_status st = sample_sizes(logits->shape[0], logits->shape[1], d);
  if (st) return st;
  if (d.rows == 0) return RTENHIP_OK;
  if (!logits->data || !uniforms || !tokens) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  if ((d.vocab > 1 && logits->strides[1] != 1) || logits->strides[0] < 0 ||
      logits->strides[0] > (int64_t(1) << 40))
    return fail(RTENHIP_UNSUPPORTED_VALUE, "Logits must have unit stride along the vocabulary");
  for (const void* p : {(const void*)logits->data, (const void*)uniforms, (const void*)tokens, (const void*)logprobs,
                        (const void*)sampling->temperatures, (const void*)sampling->top_ps,
                        (const void*)sampling->min_ps, (const void*)sampling->top_ks})
    if ((uintptr_t)p % 4) return fail(RTENHIP_UNSUPPORTED_VALUE, "Arrays must be on 4 bytes");
  if ((uintptr_t)workspace % 16) return fail(RTENHIP_UNSUPPORTED_VALUE, "Workspace must be on 16 bytes");
  const size_t need = sample_layout(d, (char*)workspace);
  if (!workspace || workspace_bytes < need) return fail(RTENHIP_INVALID_VALUE, "Workspace is too small");
  if (!ctx) return fail(RTENHIP_MISSING_INPUTS, "Missing context");
  d.logits = logits->data;
  d.row_stride = logits->strides[0];
  d.f = *sampling;
  d.uniforms = uniforms;
  d.tokens = tokens;
  d.logprobs = logprobs;
  const bool k = sampling->top_ks || (sampling->top_k > 0 && sampling->top_k < d.vocab);
  const bool p = sampling->top_ps || sampling->top_p < 1.f;
  const bool greedy = !sampling->temperatures && !(sampling->temperature > 0.f);
  if (greedy || !(k || p)) d.hist[0] = nullptr;
  if (greedy || !k) d.hist[1] = d.hist[2] = nullptr;
  if (greedy || !p) d.hist[3] = d.hist[4] = nullptr;
  DeviceScope on(reinterpret_cast<Ctx*>(ctx)->device);
  if (on.status) return on.status;
  hipStream_t s = stream_of(ctx);
  const dim3 grid((unsigned)d.rows * (unsigned)d.cuts), block(SA_THREADS);
  hipLaunchKernelGGL(sample_top_kernel, grid, block, 0, s, d);
  if (!greedy) {
    if (d.hist[0]) hipLaunchKernelGGL((sample_hist_kernel<PASS_FIRST>), grid, block, 0, s, d);
    int n = 0;
    const auto next = [&] { d.from = n ? d.states[n - 1] : nullptr, d.to = d.states[n], n++; };
    if (d.hist[1]) {
      next();
      hipLaunchKernelGGL((sample_hist_kernel<PASS_K2>), grid, block, 0, s, d);
      next();
      hipLaunchKernelGGL((sample_hist_kernel<PASS_K3>), grid, block, 0, s, d);
    }
    if (d.hist[3]) {
      next();
      hipLaunchKernelGGL((sample_hist_kernel<PASS_P2>), grid, block, 0, s, d);
      next();
      hipLaunchKernelGGL((sample_hist_kernel<PASS_P3>), grid, block, 0, s, d);
    }
    next();
    hipLaunchKernelGGL(sample_sum_kernel, grid, block, 0, s, d);
    d.from = d.to;
  }
  hipLaunchKernelGGL(sample_pick_kernel, dim3((unsigned)d.rows), block, 0, s, d);
  RTENHIP_LAUNCH_CHECK();
  return RTENHIP_OK;
}
