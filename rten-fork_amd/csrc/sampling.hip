// One token for each row of logits: temperature, top-k, top-p, min-p and a
// draw from a given random number (rtenhip_sample_f32).
//
// The token is a whole number that has to be the right one, so the weights
// m_i = exp((l_i - max) / T) are formed to 2^-31 of themselves and summed as
// integers, m_i 2^S rounded, S such that a row's sum stays below 2^63 (S = 45
// at 131,072 tokens): the sums do not depend on any order, and a draw's borders
// move by less than 2^-28 of the whole, 1/16 of a step of the random number.
//
// All filters keep a prefix of the order (falling logit, rising index), that is
// all tokens up to a last one.  It needs no sort of the row: a histogram over
// max - l in equal steps, counts and weights, leads to the bin in which the
// last one of top-k, or of top-p, lies; only the members of that bin (of the
// few bins that top-p can end in while the weight of the top-k set is not yet
// exactly known; of all bins so far if they are few) are gathered and sorted.
// Everything before them counts by its block's sum.  Rows that would gather
// more than SA_CAP tokens (equal logits, mostly) find their last one digit by
// digit instead.  The draw takes the kept weight of each block of 1024 tokens
// and one look into the block that it falls into.
//
// A row that fits a workgroup's registers takes one launch
// (sample_row_kernel).  Longer ones are cut into enough stretches to fill the
// card: with a filter a launch each for the largest logit, the histogram, the
// gathering with the blocks' sums, and the draw; without one the blocks'
// weights relative to the block's own largest, and the draw.
#include "decoder.h"

#include <algorithm>
#include <cmath>

namespace rtenhip {

constexpr int SA_BLOCK = 1024;  // tokens of a sum
constexpr int SA_EACH = SA_BLOCK / 64;
constexpr int SA_BINS = 2048;
constexpr int SA_CAP = 1024;    // gathered tokens
constexpr int SA_FEW = 128;     // up to so many are gathered rather than summed: sorted quickly
constexpr int SA_SPREAD = 256;  // threads of the kernels that cut rows
constexpr int SA_ROW = 1024;    // and of those that do not
constexpr float SA_NEG_INF = -__builtin_huge_valf();
constexpr float SA_FLT_MAX = 3.40282347e38f;

// A row's histogram: weights and counts of each bin, and of each 32 of them.
struct Hist {
  u64* mass;
  uint32_t* count;
  u64* mass32;
  uint32_t* count32;
};
constexpr size_t SA_HIST_BYTES = (SA_BINS + SA_BINS / 32) * 12;
__host__ __device__ inline Hist hist_at(void* p) {
  Hist h;
  h.mass = (u64*)p;
  h.mass32 = h.mass + SA_BINS;
  h.count = (uint32_t*)(h.mass32 + SA_BINS / 32);
  h.count32 = h.count + SA_BINS;
  return h;
}

// What the histogram says of a row: tokens of bins below `lo` are kept, those
// of lo..hi and of the bin `k` in which top-k ends are gathered, the rest is
// dropped.
struct Plan {
  int lo, hi, k;     // k = -1: top-k drops nothing
  bool p, slow;      // slow: too many to gather
  uint32_t first_k;  // gathered ones before bin k
  u64 n_lo, n_k;     // tokens before bins lo and k
  u64 m_lo, m_k, total;  // weights; total: of all tokens
};

// The same with the row's extremes, for the draw.
struct RowPlan {
  Plan plan;
  float top, least;
};

struct SampleDesc {
  const float* logits;
  int64_t row_stride;
  int rows, vocab, cuts, per_cut, blocks;  // blocks of SA_BLOCK; per_cut of them to a workgroup
  int shift;
  bool counts, masses;  // what the histograms hold
  rtenhip_sampling f;
  const float* uniforms;
  int* tokens;
  float* logprobs;
  // Workspace.
  float* cut_max;   // [rows][cuts]
  float* cut_min;   // [rows][cuts]: smallest but -infinity
  int* cut_arg;     // [rows][cuts]: first place of the largest
  u64* block_mass;  // [rows][blocks]
  float* block_max;  // [rows][blocks], without a filter
  int* block_arg;    // [rows][blocks], without a filter
  char* hist;       // [rows][cuts] of SA_HIST_BYTES
  u64* list;        // [rows][SA_CAP]
  uint32_t* listed;  // [rows]
  RowPlan* plans;    // [rows]
};

// A row's random number, brought into [0, 1).
__device__ __forceinline__ float uniform_of(const SampleDesc& d, int row) {
  const float u = d.uniforms[row];
  return !(u > 0.f) ? 0.f : u >= 1.f ? 0.99999994f : u;
}

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
  if (f.top_k >= d.vocab) f.top_k = 0;
  f.greedy = !(f.temperature > 0.f);
  return f;
}

// Falling logits, then rising indices, are rising places (56 bits); -0 is 0.
__device__ __forceinline__ u64 place_of(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t key = u & 0x80000000u ? u : ~u & 0x7fffffffu;
  return (u64)key << 24 | (uint32_t)i;
}
__device__ __forceinline__ float logit_at(u64 place) {
  const uint32_t key = (uint32_t)(place >> 24);
  return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu);
}

// ---- weights -------------------------------------------------------------------------

// 2^(j / 256) for j = 0..255 in shared memory, by the Taylor series of exp, whose
// first term left out is (ln 2)^16 / 16! < 2^-52; j 2^12 is taken off the upper
// half, and the sign flipped, for what Row::scaled adds there.
__device__ __forceinline__ void fill_powers(double* powers) {
  if (threadIdx.x < 256) {
    const double r = threadIdx.x * (0.69314718055994530942 / 256.);
    double p = 1.;
#pragma unroll
    for (int k = 15; k > 0; k--) p = __builtin_fma(p * r, 1. / k, 1.);
    powers[threadIdx.x] = __longlong_as_double(__double_as_longlong(p) + ((long long)(0x80000000u - (threadIdx.x << 12)) << 32));
  }
}

// What a row's weights and bins take.
struct Row {
  double max, scale, floor, base, min_p, inv_t;
  float half, step;
  bool infinite;
  const double* powers;
  // `max`: the largest; of a row with +infinities 0, after tame().
  // min: the smallest but -infinity, for the bins.
  __device__ Row(const Filters& f, float row_max, float row_min, int shift, const double* powers_sh) : powers(powers_sh) {
    infinite = row_max == -SA_NEG_INF;
    const float m = infinite ? 0.f : row_max;
    max = m;
    inv_t = 1. / (double)f.temperature;
    // floor * scale is -64 at every temperature, so that what is masked or no
    // number weighs nothing at an infinite one either, where any other token
    // weighs 1.
    scale = __builtin_fmax(inv_t * 1.44269504088896340736, 64e-290);
    floor = -__builtin_fmin(64. * 0.69314718055994530942 * (double)f.temperature, 1e290);
    base = 6144. + shift;
    min_p = ldexp(f.min_p > 1.f ? 1. : f.min_p > 0.f ? (double)f.min_p : 0., shift);
    // Bins reach to weights of e^-36.5 < 2^-52, less than any counts, or to
    // the smallest logit; halves, so that no difference is infinite.
    half = 0.5f * m;
    const float range = infinite ? 0.f : fminf(fminf(half - 0.5f * row_min, 18.25f * f.temperature), SA_FLT_MAX);
    step = range > 0.f ? fminf((SA_BINS - 2) / range, SA_FLT_MAX) : 0.f;
  }
  // No logit differs from the largest (or those that do weigh nothing).
  __device__ __forceinline__ bool flat() const { return step == 0.f; }
  // 0.. in falling order; SA_BINS: weighs nothing (NaN, -infinity).
  __device__ __forceinline__ int bin(float x) const {
    const float b = __builtin_fmaf(-0.5f, x, half) * step;
    return b < (float)SA_BINS ? (int)b : SA_BINS;
  }
  // 2^S exp((x - max) / T) = 2^(n + j / 256) 2^f: the exponent in fixed point,
  // 40 bits behind the point, 2048 added, is the mantissa of `y`; n and j are its
  // upper half, f < 2^-8 its lower one, whose power is 1 + q, q <= 2^-8.5 a
  // cubic in 32 bits (to 2^-31.5), the 2^-40 in its coefficients.  n is added to the exponent of 2^(j / 256).
  // (20 instructions for a token with its sum; with 26, n, the rounding and the
  // mask of `whole` a step each, a row's weights took 18,000 cycles of a CU
  // where they take 12,300.)
  __device__ __forceinline__ double scaled(float x) const {
    const double d = __builtin_fmax((double)x - max, floor);
    const u64 y = (u64)__double_as_longlong(__builtin_fma(d, scale, base));
    const uint32_t hi = (uint32_t)(y >> 32);
    const float f = (float)(uint32_t)y;
    const float q = f * __builtin_fmaf(f, __builtin_fmaf(f, 4.175665035707145e-38f, 1.9871070917790308e-25f), 6.304136882681135e-13f);
    const u64 p = (u64)__double_as_longlong(powers[hi & 255]);
    const double w = __longlong_as_double((long long)((u64)((uint32_t)(p >> 32) + (hi << 12)) << 32 | (uint32_t)p));
    return __builtin_fma(w, (double)q, w);
  }
  // Rounded to an integer m <= 2^51: the sum with 2^52 holds it in its low bits.
  __device__ __forceinline__ u64 raw(float x) const { return (u64)__double_as_longlong(scaled(x) + 4503599627370496.); }
  static __device__ __forceinline__ u64 whole(u64 raw) { return raw & 0xfffffffffffffull; }
  static __device__ __forceinline__ u64 whole_sum(u64 raws, int n) { return raws - n * 0x4330000000000000ull; }
  __device__ __forceinline__ u64 mass(float x) const { return whole(raw(x)); }
  __device__ __forceinline__ u64 mass_min(float x) const {
    const double w = scaled(x);
    return w < min_p ? 0 : whole((u64)__double_as_longlong(w + 4503599627370496.));
  }
};

// A row with +infinities: they weigh 1, the rest nothing.
__device__ __forceinline__ float tame(float x) { return x == -SA_NEG_INF ? 0.f : SA_NEG_INF; }

// ---- sums over a wave, over a workgroup ----------------------------------------------

// The largest (smallest) of the wave's, on a scalar: lanes without a neighbour
// compare with themselves.
struct Larger {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Smaller {
  __device__ float operator()(float a, float b) const { return fminf(a, b); }
  __device__ int operator()(int a, int b) const { return min(a, b); }
};
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T own_dpp(T x) {
  const int i = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xf, false));
}
template <typename Op, typename T>
__device__ __forceinline__ T row_best(T x) {  // of a row of 16 lanes, on its last
  const Op op;
  x = op(x, own_dpp<0x111, 0xf>(x));
  x = op(x, own_dpp<0x112, 0xf>(x));
  x = op(x, own_dpp<0x114, 0xf>(x));
  return op(x, own_dpp<0x118, 0xf>(x));
}
template <typename T>
__device__ __forceinline__ T scalar(T x, int lane) {
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
template <typename Op, typename T>
__device__ __forceinline__ T wave_best(T x) {
  const Op op;
  x = row_best<Op>(x);
  x = op(x, own_dpp<0x142, 0xa>(x));
  x = op(x, own_dpp<0x143, 0xc>(x));
  return scalar(x, 63);
}

// Exclusive prefix over the SA_ROW threads; `all` is the sum.
__device__ __forceinline__ u64 block_scan(u64 x, u64* sh, u64& all) {
  static_assert(SA_ROW == 16 * 64, "a wave's sum to each lane of a row");
  const u64 in = wave_scan(x);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[wave] = in;
  __syncthreads();
  const u64 own = sh[threadIdx.x & 15];
  const u64 s = row_scan(own);
  all = lane_of(s, 15);
  return in - x + lane_of(s - own, __builtin_amdgcn_readfirstlane(wave));
}

// Largest of a, smallest of b over the workgroup.
template <int NT>
__device__ __forceinline__ void block_extremes(float& a, float& b, float* sh) {
  a = wave_best<Larger>(a), b = wave_best<Smaller>(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a, sh[16 + (threadIdx.x >> 6)] = b;
  __syncthreads();
  a = scalar(row_best<Larger>(sh[threadIdx.x % (NT / 64)]), 15);
  b = scalar(row_best<Smaller>(sh[16 + threadIdx.x % (NT / 64)]), 15);
}
template <int NT>
__device__ __forceinline__ int block_least(int a, int* sh) {
  a = wave_best<Smaller>(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
  __syncthreads();
  return scalar(row_best<Smaller>(sh[threadIdx.x % (NT / 64)]), 15);
}

// ---- tokens --------------------------------------------------------------------------

// A block's tokens, lane l those at 4 l .. 4 l + 3, 256 + 4 l, ...: loads of 16
// bytes, at any address of a float, but for a row's last block.
__device__ __forceinline__ int token_of(int b, int u) {
  return b * SA_BLOCK + u / 4 * 256 + (int)(threadIdx.x & 63) * 4 + u % 4;
}
typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void load_block(const float* x, int vocab, int b, float (&v)[SA_EACH]) {
  if ((b + 1) * SA_BLOCK <= vocab) {
#pragma unroll
    for (int u = 0; u < SA_EACH; u += 4) {
      const Float4 four = *(const Float4*)(x + token_of(b, u));
      v[u] = four[0], v[u + 1] = four[1], v[u + 2] = four[2], v[u + 3] = four[3];
    }
  } else {
#pragma unroll
    for (int u = 0; u < SA_EACH; u++) v[u] = x[min(token_of(b, u), vocab - 1)];
  }
}
__device__ __forceinline__ void end_block(int vocab, int b, float (&v)[SA_EACH]) {
  if ((b + 1) * SA_BLOCK > vocab) {
#pragma unroll
    for (int u = 0; u < SA_EACH; u++)
      if (token_of(b, u) >= vocab) v[u] = SA_NEG_INF;
  }
}

// Calls g(b, v) for this wave's blocks of a stretch in memory; v is -infinity
// past the row's end.  Ahead: the first block is on its way from the start, the
// next one during each g.
struct Ahead {
  const float* x;
  int vocab, b0, b1;
  float first[SA_EACH];
  __device__ __forceinline__ Ahead(const float* row, int length, int from, int to)
      : x(row), vocab(length), b0(from + (int)(threadIdx.x >> 6)), b1(to) {
    load_block(x, vocab, min(b0, b1 - 1), first);
  }
  template <typename G>
  __device__ __forceinline__ void blocks(bool infinite, G g) const {
    float v[SA_EACH], next[SA_EACH];
    for (int u = 0; u < SA_EACH; u++) v[u] = first[u];
    for (int b = b0; b < b1; b += SA_SPREAD / 64) {
      const bool more = b + SA_SPREAD / 64 < b1;
      if (more) load_block(x, vocab, b + SA_SPREAD / 64, next);
      end_block(vocab, b, v);
      if (infinite) {
#pragma unroll
        for (int u = 0; u < SA_EACH; u++) v[u] = tame(v[u]);
      }
      g(b, v);
      if (!more) break;
      for (int u = 0; u < SA_EACH; u++) v[u] = next[u];
    }
  }
};
struct Whole {
  const float* x;
  int vocab, count;
  template <typename G>
  __device__ __forceinline__ void blocks(bool infinite, G g) const {
    for (int b = (int)(threadIdx.x >> 6); b < count; b += SA_ROW / 64) {
      float v[SA_EACH];
      load_block(x, vocab, b, v);
      end_block(vocab, b, v);
      if (infinite) {
#pragma unroll
        for (int u = 0; u < SA_EACH; u++) v[u] = tame(v[u]);
      }
      g(b, v);
    }
  }
};

// A row in a workgroup's registers.
template <int K>
struct Held {
  float (&v)[K][SA_EACH];
  int count;
  template <typename G>
  __device__ __forceinline__ void blocks(bool, G g) const {  // (tamed already)
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int b = (int)(threadIdx.x >> 6) + k * (SA_ROW / 64);
      if (b < count) g(b, v[k]);
    }
  }
};

// ---- histograms ----------------------------------------------------------------------

template <int NT>
__device__ __forceinline__ void clear_hist(const Hist& h) {
  for (int i = threadIdx.x; i < SA_BINS; i += NT) h.mass[i] = 0, h.count[i] = 0;
}

// All tokens into the bins of their distance from the largest.
template <typename S>
__device__ __forceinline__ void fill_hist(const S& src, const Row& r, bool counts, bool masses, const Hist& h) {
  src.blocks(r.infinite, [&](int, const float (&v)[SA_EACH]) {
#pragma unroll
    for (int u = 0; u < SA_EACH; u++) {
      const int bin = r.bin(v[u]);
      if (bin < SA_BINS) {
        if (counts) atomicAdd(&h.count[bin], 1u);
        if (masses) atomicAdd(&h.mass[bin], r.mass(v[u]));
      }
    }
  });
}

// Calls f(bin, mass, count) for all bins, a lane each, and f32(i, mass, count)
// with the sums of each 32.
template <int NT, typename F, typename F32>
__device__ __forceinline__ void sum_hist(const Hist& h, F f, F32 f32) {
#pragma unroll
  for (int bin = threadIdx.x; bin < SA_BINS; bin += NT) {
    u64 m = h.mass[bin];
    uint32_t c = h.count[bin];
    f(bin, m, c);
    m = half_scan(m), c = half_scan(c);
    if (threadIdx.x % 32 == 31) f32(bin / 32, m, c);
  }
}

// The bin at which the counts (weights) from the first on reach `target` >= 1;
// what is before it and in it.  Whole waves call it.
struct Found {
  int bin;  // -1: all of them are less
  u64 count, mass, in_count, in_mass;
};
struct OneHist {
  Hist h;
  bool counts, masses;
  __device__ __forceinline__ void bins32(int i, uint32_t& c, u64& m) const {
    c = counts ? h.count32[i] : 0, m = masses ? h.mass32[i] : 0;
  }
  __device__ __forceinline__ void bins(int i, uint32_t& c, u64& m) const {
    c = counts ? h.count[i] : 0, m = masses ? h.mass[i] : 0;
  }
};
// Of a row cut into stretches: the sums of theirs.
struct CutHists {
  const char* first;
  int cuts;
  bool counts, masses;
  __device__ __forceinline__ void sum(size_t count_at, size_t mass_at, int i, uint32_t& c, u64& m) const {
    c = 0, m = 0;
    const uint32_t* cp = (const uint32_t*)(first + count_at) + i;
    const u64* mp = (const u64*)(first + mass_at) + i;
    for (int k0 = 0; k0 < cuts; k0 += 16) {  // (the loads of 16 at once, the last one's again past the end)
      if (counts) {
        uint32_t in[16];
#pragma unroll
        for (int k = 0; k < 16; k++) in[k] = cp[min(k0 + k, cuts - 1) * (SA_HIST_BYTES / 4)];
#pragma unroll
        for (int k = 0; k < 16; k++) c += k0 + k < cuts ? in[k] : 0;
      }
      if (masses) {
        u64 in[16];
#pragma unroll
        for (int k = 0; k < 16; k++) in[k] = mp[min(k0 + k, cuts - 1) * (SA_HIST_BYTES / 8)];
#pragma unroll
        for (int k = 0; k < 16; k++) m += k0 + k < cuts ? in[k] : 0;
      }
    }
  }
  __device__ __forceinline__ void bins32(int i, uint32_t& c, u64& m) const {
    sum((SA_BINS + SA_BINS / 32) * 8 + SA_BINS * 4, SA_BINS * 8, i, c, m);
  }
  __device__ __forceinline__ void bins(int i, uint32_t& c, u64& m) const { sum((SA_BINS + SA_BINS / 32) * 8, 0, i, c, m); }
};
// Each 32 bins' counts and weights with those before them, a lane each.
template <typename H>
struct Bins {
  const H h;
  uint32_t c, cs;
  u64 m, ms;
  __device__ __forceinline__ Bins(const H& hist) : h(hist) {
    h.bins32(threadIdx.x & 63, c, m);
    cs = h.counts ? wave_scan(c) : 0;
    ms = h.masses ? wave_scan(m) : 0;
  }
  __device__ __forceinline__ u64 all_mass() const { return lane_of(ms, 63); }
  __device__ __forceinline__ Found find(bool by_mass, u64 target) const {
    const int lane = threadIdx.x & 63;
    Found r;
    u64 hit = __ballot((by_mass ? ms : (u64)cs) >= target);
    if (!hit) {
      r.bin = -1, r.count = lane_of(cs, 63), r.mass = all_mass(), r.in_count = r.in_mass = 0;
      return r;
    }
    const int g = __builtin_ctzll(hit);
    uint32_t n;
    u64 w;
    h.bins(g * 32 + (lane & 31), n, w);
    if (lane >= 32) n = 0, w = 0;
    const uint32_t ns = lane_of(cs - c, g) + (h.counts ? wave_scan(n) : 0);
    const u64 ws = lane_of(ms - m, g) + (h.masses ? wave_scan(w) : 0);
    hit = __ballot((by_mass ? ws : (u64)ns) >= target);
    const int b = __builtin_ctzll(hit);
    r.bin = g * 32 + b;
    r.in_count = lane_of(n, b), r.in_mass = lane_of(w, b);
    r.count = lane_of(ns, b) - r.in_count, r.mass = lane_of(ws, b) - r.in_mass;
    return r;
  }
};

// ceil(share of the kept weight), at least 1 so that the first token stays.
__device__ __forceinline__ u64 p_target(float p, u64 total) {
  const double t = __builtin_ceil((p > 0.f ? (double)p : 0.) * (double)total);
  const u64 n = (u64)t;
  return n < 1 ? 1 : n > total ? total : n;
}

template <typename H>
__device__ __forceinline__ Plan plan_of(const Bins<H>& bins, const Row& r, const Filters& f) {
  const bool masses = bins.h.masses, counts = bins.h.counts;
  Plan q{};
  q.lo = SA_BINS, q.hi = q.k = -1;
  q.p = f.top_p < 1.f;
  if (!(f.top_k > 0) && !q.p) return q;
  if (r.flat()) {
    q.slow = true;
    return q;
  }
  Found a{};
  if (f.top_k > 0) {
    a = bins.find(false, (u64)f.top_k);
    q.k = a.bin, q.n_k = a.count, q.m_k = a.mass, q.total = a.mass;
  }
  if (q.k < 0 && !q.p) return q;
  u64 n_hi;  // tokens up to bin hi
  if (q.k >= 0 && (!q.p || a.count + a.in_count <= (masses ? SA_FEW : SA_CAP))) {
    q.lo = q.hi = q.k;
    q.n_lo = a.count, q.m_lo = a.mass, n_hi = a.count + a.in_count;
  } else if (!masses) {
    q.slow = true;
    return q;
  } else {
    if (q.k < 0) q.total = bins.all_mass();
    const Found b = bins.find(true, p_target(f.top_p, q.k < 0 ? q.total : a.mass));
    q.lo = q.hi = b.bin;
    q.n_lo = b.count, q.m_lo = b.mass, n_hi = b.count + b.in_count;
    if (q.k >= 0) {
      const Found c = bins.find(true, p_target(f.top_p, a.mass + a.in_mass));
      q.hi = c.bin, n_hi = c.count + c.in_count;
    }
  }
  if (counts && n_hi <= (masses || !q.p ? SA_FEW : SA_CAP)) q.lo = 0, q.n_lo = q.m_lo = 0;
  u64 n = n_hi - q.n_lo;
  if (q.k > q.hi) q.first_k = (uint32_t)n, n += a.in_count;
  else if (q.k >= 0) q.first_k = (uint32_t)(q.n_k - q.n_lo);
  q.slow = n > SA_CAP;  // (without counts only the gathering shows it)
  return q;
}

// A wave's tokens of a block that may be kept.
struct Few {
  float x[SA_BLOCK];
  uint16_t i[SA_BLOCK];
};

// Tokens to gather into list[0..], and each block's kept weight before them.
// The few tokens that the filters leave are moved together first: spread over
// a block they would take as many steps as all.
template <typename S>
__device__ __forceinline__ void gather(const S& src, const Row& r, const Plan& q, Few& few, u64* list,
                                       uint32_t* listed, u64* block_mass) {
  const int lane = threadIdx.x & 63;
  // No logit below `least` is in any of the bins: twice the two roundings of a
  // bin's number are taken off.
  const int end = q.lo == SA_BINS ? SA_BINS : max(q.hi, q.k) + 1;
  const float least = r.flat() ? SA_NEG_INF : (float)(r.max - 2.000001 * end / (double)r.step);
  src.blocks(r.infinite, [&](int b, const float (&v)[SA_EACH]) {
    u64 mass = 0;
    if (q.lo == SA_BINS) {
#pragma unroll
      for (int u = 0; u < SA_EACH; u++) mass += r.mass_min(v[u]);
    } else {
      uint32_t n = 0;
#pragma unroll
      for (int u = 0; u < SA_EACH; u++) {
        const bool in = v[u] >= least;
        const u64 lanes = __ballot(in);
        const uint32_t at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
        if (in) few.x[at] = v[u], few.i[at] = (uint16_t)token_of(0, u);
        n += __builtin_popcountll(lanes);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (uint32_t j = lane; j < n; j += 64) {
        const float x = few.x[j];
        const int bin = r.bin(x);
        if (bin < q.lo) {
          mass += r.mass_min(x);
        } else if (bin <= q.hi || bin == q.k) {
          const uint32_t at = atomicAdd(listed, 1u);
          if (at < SA_CAP) list[at] = place_of(x, b * SA_BLOCK + few.i[j]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (q.lo) mass = wave_sum(mass);
    if (lane == 0) block_mass[b] = mass;
  });
}

// Sorts n <= SA_CAP different numbers in shared memory: each goes to the place
// that the number of smaller ones says, which the 16 lanes of a row count.  (A
// bitonic network's steps wait for one another: sorting 64 with the rest of
// `resolve` took 12,500 cycles and takes 3,500 this way.)
__device__ __forceinline__ void sort_list(const u64* list, u64* sorted, int n) {
  const int part = threadIdx.x & 15;
  for (int e = threadIdx.x >> 4; e - (int)(threadIdx.x >> 4) < n; e += SA_ROW / 16) {
    const u64 own = e < n ? list[e] : 0;
    uint32_t smaller = 0;
    for (int j = part; j < n; j += 16) smaller += list[j] < own;
    smaller = row_scan(smaller);
    if (part == 15 && e < n) sorted[smaller] = own;
  }
  __syncthreads();
}

struct SampleShared {
  u64 scan[SA_ROW / 64];
  float extremes[32];
  int least[SA_ROW / 64];
  u64 limit, base;
  int block;
  uint32_t listed;
};

// The last place that is kept, from the n gathered tokens; what they add to
// their blocks.
template <bool LOCAL>
__device__ __forceinline__ u64 resolve(const u64* list, u64* sorted, int n, const Row& r, const Filters& f,
                                       const Plan& q, u64* block_mass, SampleShared& sh) {
  static_assert(SA_CAP == SA_ROW, "one to each thread");
  if (!n) return ~0ull;
  if (threadIdx.x == 0) sh.limit = 0;
  sort_list(list, sorted, n);
  const int at = threadIdx.x;
  const u64 place = at < n ? sorted[at] : ~0ull;
  const float x = logit_at(place);
  const int bin = at < n ? r.bin(x) : SA_BINS;
  const u64 rank = bin == q.k ? q.n_k + at - q.first_k : q.n_lo + at;
  const bool in_k = at < n && (q.k < 0 || rank < (u64)f.top_k);
  const u64 mass = in_k ? r.mass(x) : 0;
  bool kept = in_k && bin <= q.hi;
  if (q.p) {
    u64 total = q.total, all;
    const u64 before = q.m_lo + block_scan(bin <= q.hi ? mass : 0, sh.scan, all);
    if (q.k >= 0) {
      if (q.lo == 0 && q.hi == q.k) {
        total = all;
      } else {
        block_scan(bin == q.k ? mass : 0, sh.scan, all);
        total = q.m_k + all;
      }
    }
    kept = kept && before < p_target(f.top_p, total);
  }
  if (kept) {
    const u64 m = r.mass_min(x);
    u64* to = &block_mass[(place & 0xffffff) / SA_BLOCK];
    if (m) {
      if (LOCAL)
        atomicAdd(to, m);
      else
        __hip_atomic_fetch_add(to, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // The kept ones are the first: the last of a wave's, the largest of those.
  const u64 lanes = __ballot(kept);
  if (lanes) {
    const u64 last = lane_of(place, 63 - __builtin_clzll(lanes));
    if ((threadIdx.x & 63) == 0) atomicMax(&sh.limit, last);
  }
  __syncthreads();
  return sh.limit;  // (the first gathered one is always kept)
}

// ---- digit by digit ------------------------------------------------------------------

// The place up to which tokens with places <= bound count `target`, or weigh
// the share p of all of them: five digits of 11 bits and one of 1.
__device__ __forceinline__ u64 select_place(const Whole& src, const Row& r, const Hist& h, bool by_mass, u64 target,
                                            float p, u64 bound) {
  const int lane = threadIdx.x & 63;
  u64 prefix = 0;
  for (int shift = 45; shift >= 0; shift = shift > 11 ? shift - 11 : shift - 1) {
    const int bits = shift ? 11 : 1;
    __syncthreads();
    clear_hist<SA_ROW>(h);
    __syncthreads();
    src.blocks(r.infinite, [&](int b, const float (&v)[SA_EACH]) {
#pragma unroll 1
      for (int u = 0; u < SA_EACH; u++) {
        float x = v[0];
#pragma unroll
        for (int w = 1; w < SA_EACH; w++) x = w == u ? v[w] : x;
        const u64 place = place_of(x, token_of(b, u));
        const bool in = r.bin(x) < SA_BINS && place <= bound && place >> shift >> bits == prefix;
        const u64 lanes = __ballot(in);
        if (!lanes) continue;
        const int bin = (int)(place >> shift) & ((1 << bits) - 1);
        u64 mass = in && by_mass ? r.mass(x) : 0;
        // Equal logits share all digits but the last two.
        if (__ballot(in && bin == __builtin_amdgcn_readlane(bin, __builtin_ctzll(lanes))) == lanes) {
          mass = wave_sum(mass);
          if (lane == __builtin_ctzll(lanes)) {
            atomicAdd(&h.count[bin], (uint32_t)__builtin_popcountll(lanes));
            atomicAdd(&h.mass[bin], mass);
          }
        } else if (in) {
          atomicAdd(&h.count[bin], 1u);
          atomicAdd(&h.mass[bin], mass);
        }
      }
    });
    __syncthreads();
    sum_hist<SA_ROW>(
        h, [](int, u64, uint32_t) {}, [&](int i, u64 m, uint32_t c) { h.mass32[i] = m, h.count32[i] = c; });
    __syncthreads();
    const Bins<OneHist> bins(OneHist{h, true, by_mass});
    if (by_mass && shift == 45) target = p_target(p, bins.all_mass());
    const Found a = bins.find(by_mass, target);
    if (a.bin < 0) return bound;
    target -= by_mass ? a.mass : a.count;
    prefix = prefix << bits | (u64)a.bin;
  }
  return prefix;
}

// The last place that is kept, and the blocks' weights.
__device__ __forceinline__ u64 select_row(const Whole& src, const Row& r, const Filters& f, const Hist& h,
                                          u64* block_mass) {
  const int lane = threadIdx.x & 63;
  u64 limit = ~0ull;
  if (f.top_k > 0) limit = select_place(src, r, h, false, (u64)f.top_k, 1.f, limit);
  if (f.top_p < 1.f) limit = select_place(src, r, h, true, 1, f.top_p, limit);
  src.blocks(r.infinite, [&](int b, const float (&v)[SA_EACH]) {
    u64 mass = 0;
#pragma unroll
    for (int u = 0; u < SA_EACH; u++)
      if (place_of(v[u], token_of(b, u)) <= limit) mass += r.mass_min(v[u]);
    mass = wave_sum(mass);
    if (lane == 0) block_mass[b] = mass;
  });
  __syncthreads();
  return limit;
}

// ---- the draw ------------------------------------------------------------------------

// The block from its weights weight_of(b), then the token in it.  RELATIVE: the
// block's tokens by `of_block(b)`, weights relative to the block's largest.
template <bool RELATIVE, typename W, typename B>
__device__ __forceinline__ void draw(const SampleDesc& d, int row, float u, const Row& r, bool infinite, u64 limit,
                                     W weight_of, B of_block, SampleShared& sh) {
  const int tid = threadIdx.x;
  const int each = (d.blocks + SA_ROW - 1) / SA_ROW;
  const int b0 = min(d.blocks, tid * each), b1 = min(d.blocks, b0 + each);
  u64 mass = 0, total, all;
  for (int b = b0; b < b1; b++) mass += weight_of(b);
  u64 at = block_scan(mass, sh.scan, total);
  u64 left = (u64)((double)u * (double)total);
  left = min(left, total - 1);
  if (left >= at && left < at + mass) {
    for (int b = b0; b < b1; b++) {
      const u64 m = weight_of(b);
      if (left < at + m) {
        sh.block = b, sh.base = at, sh.limit = m;
        break;
      }
      at += m;
    }
  }
  __syncthreads();
  static_assert(SA_BLOCK == SA_ROW, "a token to each thread");
  const int b = sh.block, i = b * SA_BLOCK + tid;
  float x = d.logits[(int64_t)row * d.row_stride + min(i, d.vocab - 1)];
  if (i >= d.vocab) x = SA_NEG_INF;
  if (infinite) x = tame(x);
  left -= sh.base;
  if constexpr (RELATIVE) {
    mass = of_block(b).mass(x);
  } else {
    mass = place_of(x, i) <= limit ? r.mass_min(x) : 0;
  }
  at = block_scan(mass, sh.scan, all);
  if (RELATIVE) left = (u64)((double)left * ((double)all / (double)sh.limit));
  left = min(left, all - 1);
  if (left >= at && left < at + mass) {
    d.tokens[row] = i;
    if (d.logprobs) d.logprobs[row] = (float)(((double)x - r.max) * r.inv_t - log((double)total * ldexp(1., -d.shift)));
  }
}

__device__ __forceinline__ void no_token(const SampleDesc& d, int row) {
  d.tokens[row] = -1;
  if (d.logprobs) d.logprobs[row] = SA_NEG_INF;
}
__device__ __forceinline__ void sure_token(const SampleDesc& d, int row, int token) {
  d.tokens[row] = token;
  if (d.logprobs) d.logprobs[row] = 0.f;
}

// ---- kernels: a row to a workgroup ---------------------------------------------------

// Bound by one CU: 122 KB of logits take it 2.7 us to arrive, and every pass over
// 30 tokens a thread is 1 us and more.  One row of 30,522, all filters: 11 us;
// 256 rows of 32,768 with top-p: 22 us.
template <int K>
__global__ __launch_bounds__(SA_ROW) void sample_row_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ double powers[256];
  __shared__ Few few[SA_ROW / 64];
  __shared__ u64 list[SA_CAP], sorted[SA_CAP], block_mass[K * SA_ROW / 64];
  __shared__ u64 hist_sh[SA_HIST_BYTES / 8];
  const Hist h = hist_at(hist_sh);
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const float* x = d.logits + (int64_t)row * d.row_stride;
  const Filters f = filters_of(d, row);
  const float u = uniform_of(d, row);
  float v[K][SA_EACH];
#pragma unroll
  for (int k = 0; k < K; k++) load_block(x, d.vocab, min(wave + k * (SA_ROW / 64), d.blocks - 1), v[k]);
  fill_powers(powers);
  const bool filter = f.top_k > 0 || f.top_p < 1.f;
  if (filter) clear_hist<SA_ROW>(h);
  if (tid == 0) sh.listed = 0;
  const Held<K> src{v, d.blocks};
  float top = SA_NEG_INF, least = -SA_NEG_INF;
#pragma unroll
  for (int k = 0; k < K; k++) {
    end_block(d.vocab, wave + k * (SA_ROW / 64), v[k]);
#pragma unroll
    for (int u = 0; u < SA_EACH; u++) {
      top = fmaxf(top, v[k][u]);
      least = fminf(least, v[k][u] > SA_NEG_INF ? v[k][u] : least);
    }
  }
  block_extremes<SA_ROW>(top, least, sh.extremes);
  if (top == SA_NEG_INF) {
    if (tid == 0) no_token(d, row);
    return;
  }
  if (f.greedy) {
    int arg = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int u = 0; u < SA_EACH; u++)
        if (v[k][u] == top) arg = min(arg, token_of(wave + k * (SA_ROW / 64), u));
    arg = block_least<SA_ROW>(arg, sh.least);
    if (tid == 0) sure_token(d, row, arg);
    return;
  }
  const bool infinite = top == -SA_NEG_INF;
  if (infinite) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int u = 0; u < SA_EACH; u++) v[k][u] = tame(v[k][u]);
  }
  const Row r(f, top, least, d.shift, powers);
  Plan q;
  if (f.top_k > 0 && f.top_k <= SA_ROW / 16 && !r.flat()) {
    // A few: the threads' largest ones alone have top_k in the bins up to some
    // one, so all of the top_k are in these bins, and not many more are.  (For
    // more than 1 / 16 of the threads too many more are: with 30,522 tokens
    // top-50 took 12 us by the histogram of all and takes 10.7, top-256 took 16
    // this way and takes 14.)
    float own = SA_NEG_INF;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int u = 0; u < SA_EACH; u++) own = fmaxf(own, v[k][u]);
    const int bin = r.bin(own);
    if (bin < SA_BINS) atomicAdd(&h.count[bin], 1u);
    __syncthreads();
    sum_hist<SA_ROW>(
        h, [](int, u64, uint32_t) {}, [&](int i, u64, uint32_t c) { h.count32[i] = c; });
    __syncthreads();
    const Found a = Bins<OneHist>(OneHist{h, true, false}).find(false, (u64)f.top_k);
    q = Plan{};
    q.hi = q.k = a.bin < 0 ? SA_BINS - 1 : a.bin;
    q.p = f.top_p < 1.f;
  } else {
    if (filter && !r.flat()) {
      fill_hist(src, r, d.counts, d.masses, h);
      __syncthreads();
      sum_hist<SA_ROW>(
          h, [](int, u64, uint32_t) {}, [&](int i, u64 m, uint32_t c) { h.mass32[i] = m, h.count32[i] = c; });
      __syncthreads();
    }
    q = plan_of(Bins<OneHist>(OneHist{h, d.counts, d.masses}), r, f);
  }
  if (!q.slow) {
    gather(src, r, q, few[tid >> 6], list, &sh.listed, block_mass);
    __syncthreads();
    q.slow = sh.listed > SA_CAP;
  }
  u64 limit;
  if (q.slow) {
    // (From memory again: the passes would keep too much beside the tokens.)
    limit = select_row(Whole{x, d.vocab, d.blocks}, r, f, h, block_mass);
  } else {
    limit = resolve<true>(list, sorted, (int)sh.listed, r, f, q, block_mass, sh);
  }
  draw<false>(
      d, row, u, r, infinite, limit, [&](int b) { return block_mass[b]; }, [](int) {}, sh);
}

// ---- kernels: rows cut into stretches ------------------------------------------------

// A workgroup's row and stretch.
struct Cut {
  int row, b0, b1;
  const float* x;
  __device__ Cut(const SampleDesc& d) {
    row = blockIdx.x / d.cuts;
    const int cut = blockIdx.x - row * d.cuts;
    b0 = cut * d.per_cut, b1 = min(d.blocks, b0 + d.per_cut);
    x = d.logits + (int64_t)row * d.row_stride;
  }
  __device__ __forceinline__ Ahead stretch(const SampleDesc& d) const { return Ahead(x, d.vocab, b0, b1); }
};

// The four kernels for 64 rows of 100,003 with top-p, 25.6 MB that stay in the
// caches: 8, 14, 13 and 6 us.  Each is a launch, some reductions over the row
// that every workgroup repeats (the first tokens on their way meanwhile), and
// one pass; 5 us would be the reading at a copy's rate.

// Largest logit with its first place, and smallest, of each stretch.
__global__ __launch_bounds__(SA_SPREAD) void sample_top_kernel(SampleDesc d) {
  __shared__ float extremes[32];
  __shared__ int least_sh[SA_SPREAD / 64];
  const Cut c(d);
  const int tid = threadIdx.x;
  if (c.b0 == 0 && tid == 0) d.listed[c.row] = 0;
  float top = SA_NEG_INF, least = -SA_NEG_INF;
  int arg = 0x7fffffff;
  c.stretch(d).blocks(false, [&](int b, const float (&v)[SA_EACH]) {
#pragma unroll
    for (int u = 0; u < SA_EACH; u++) {
      if (v[u] > top) top = v[u], arg = token_of(b, u);  // (never for a NaN)
      least = fminf(least, v[u] > SA_NEG_INF ? v[u] : least);
    }
  });
  const float own = top;
  block_extremes<SA_SPREAD>(top, least, extremes);
  arg = block_least<SA_SPREAD>(own == top ? arg : 0x7fffffff, least_sh);
  if (tid == 0) d.cut_max[blockIdx.x] = top, d.cut_min[blockIdx.x] = least, d.cut_arg[blockIdx.x] = arg;
}

// A row's largest and smallest from its stretches'.
template <int NT>
__device__ __forceinline__ void row_extremes(const SampleDesc& d, int row, float& top, float& least, float* sh) {
  top = SA_NEG_INF, least = -SA_NEG_INF;
  for (int i = threadIdx.x; i < d.cuts; i += NT)
    top = fmaxf(top, d.cut_max[row * d.cuts + i]), least = fminf(least, d.cut_min[row * d.cuts + i]);
  block_extremes<NT>(top, least, sh);
}

__global__ __launch_bounds__(SA_SPREAD) void sample_hist_kernel(SampleDesc d) {
  __shared__ float extremes[32];
  __shared__ double powers[256];
  __shared__ u64 hist_sh[SA_HIST_BYTES / 8];
  const Hist h = hist_at(hist_sh);
  const Cut c(d);
  const Ahead src = c.stretch(d);
  const Filters f = filters_of(d, c.row);
  fill_powers(powers);
  clear_hist<SA_SPREAD>(h);
  float top, least;
  row_extremes<SA_SPREAD>(d, c.row, top, least, extremes);
  if (f.greedy || top == SA_NEG_INF) return;
  const Row r(f, top, least, d.shift, powers);
  if (r.flat()) return;
  fill_hist(src, r, d.counts, d.masses, h);
  __syncthreads();
  const Hist to = hist_at(d.hist + (size_t)blockIdx.x * SA_HIST_BYTES);
  sum_hist<SA_SPREAD>(
      h,
      [&](int bin, u64 m, uint32_t n) {
        if (d.counts) to.count[bin] = n;
        if (d.masses) to.mass[bin] = m;
      },
      [&](int i, u64 m, uint32_t n) {
        if (d.counts) to.count32[i] = n;
        if (d.masses) to.mass32[i] = m;
      });
}

__global__ __launch_bounds__(SA_SPREAD) void sample_gather_kernel(SampleDesc d) {
  __shared__ float extremes[32];
  __shared__ double powers[256];
  __shared__ Few few[SA_SPREAD / 64];
  __shared__ u64 list[SA_CAP];
  __shared__ uint32_t listed, base;
  const Cut c(d);
  const Ahead src = c.stretch(d);
  const Filters f = filters_of(d, c.row);
  // (Also on its way meanwhile; nothing of it is used where there is none.)
  const Bins<CutHists> bins(
      CutHists{d.hist + (size_t)c.row * d.cuts * SA_HIST_BYTES, d.cuts, d.hist && d.counts, d.hist && d.masses});
  fill_powers(powers);
  if (threadIdx.x == 0) listed = 0;
  float top, least;
  row_extremes<SA_SPREAD>(d, c.row, top, least, extremes);
  const bool last = f.greedy || top == SA_NEG_INF;
  const Row r(f, top, least, d.shift, powers);
  const Plan q = last ? Plan{} : plan_of(bins, r, f);
  if (c.b0 == 0 && threadIdx.x == 0) d.plans[c.row] = RowPlan{q, top, least};
  if (last) return;
  if (q.slow) return;
  gather(src, r, q, few[threadIdx.x >> 6], list, &listed, d.block_mass + (int64_t)c.row * d.blocks);
  __syncthreads();
  const uint32_t n = listed;
  if (!n) return;
  if (threadIdx.x == 0) base = atomicAdd(&d.listed[c.row], n);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n && base + i < SA_CAP; i += SA_SPREAD)
    d.list[(int64_t)c.row * SA_CAP + base + i] = list[i];
}

__global__ __launch_bounds__(SA_ROW) void sample_pick_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ double powers[256];
  __shared__ u64 list[SA_CAP], sorted[SA_CAP];
  __shared__ u64 hist_sh[SA_HIST_BYTES / 8];
  const int row = blockIdx.x, tid = threadIdx.x;
  const Filters f = filters_of(d, row);
  const float u = uniform_of(d, row);
  fill_powers(powers);
  const RowPlan known = d.plans[row];
  const uint32_t n = d.listed[row];
  const float top = known.top;
  __syncthreads();
  if (top == SA_NEG_INF) {
    if (tid == 0) no_token(d, row);
    return;
  }
  if (f.greedy) {
    int arg = 0x7fffffff;
    for (int i = tid; i < d.cuts; i += SA_ROW)
      if (d.cut_max[row * d.cuts + i] == top) arg = min(arg, d.cut_arg[row * d.cuts + i]);
    arg = block_least<SA_ROW>(arg, sh.least);
    if (tid == 0) sure_token(d, row, arg);
    return;
  }
  const bool infinite = top == -SA_NEG_INF;
  const Row r(f, top, known.least, d.shift, powers);
  const Plan q = known.plan;
  u64* block_mass = d.block_mass + (int64_t)row * d.blocks;
  u64 limit;
  if (q.slow || n > SA_CAP) {
    const Whole src{d.logits + (int64_t)row * d.row_stride, d.vocab, d.blocks};
    limit = select_row(src, r, f, hist_at(hist_sh), block_mass);
  } else {
    for (int i = tid; i < (int)n; i += SA_ROW) list[i] = d.list[(int64_t)row * SA_CAP + i];
    __syncthreads();
    limit = resolve<false>(list, sorted, (int)n, r, f, q, block_mass, sh);
  }
  draw<false>(
      d, row, u, r, infinite, limit,
      [&](int b) { return __hip_atomic_load(&block_mass[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }, [](int) {},
      sh);
}

// Without a filter: a block's largest logit, its first place, and the block's
// weight relative to it in units of 2^-50, by a wave that holds the block.
// Bound by memory: 256 rows of 131,072, 134 MB, in 30 us, 4.5 TB/s (a copy: 4.7).
constexpr int SA_BLOCK_SHIFT = 50;
__global__ __launch_bounds__(SA_SPREAD) void sample_block_kernel(SampleDesc d) {
  __shared__ double powers[256];
  const Cut c(d);
  const Filters f = filters_of(d, c.row);
  const int lane = threadIdx.x & 63;
  fill_powers(powers);
  __syncthreads();
  Row r(f, 0.f, 0.f, SA_BLOCK_SHIFT, powers);
  c.stretch(d).blocks(false, [&](int b, const float (&v)[SA_EACH]) {
    float m = SA_NEG_INF;
#pragma unroll
    for (int u = 0; u < SA_EACH; u++) m = fmaxf(m, v[u]);
    m = wave_best<Larger>(m);
    int arg = 0x7fffffff;
    u64 mass = 0;
    if (f.greedy) {
#pragma unroll
      for (int u = SA_EACH - 1; u >= 0; u--)
        if (v[u] == m) arg = token_of(b, u);
      arg = wave_best<Smaller>(arg);
    } else if (m > SA_NEG_INF) {
      r.max = m == -SA_NEG_INF ? 0. : m;
      if (m == -SA_NEG_INF) {
#pragma unroll
        for (int u = 0; u < SA_EACH; u++) mass += r.raw(tame(v[u]));
      } else {
#pragma unroll
        for (int u = 0; u < SA_EACH; u++) mass += r.raw(v[u]);
      }
      mass = wave_sum(Row::whole_sum(mass, SA_EACH));
    }
    if (lane == 0) {
      const int64_t at = (int64_t)c.row * d.blocks + b;
      d.block_max[at] = m;
      d.block_arg[at] = arg;
      d.block_mass[at] = mass;
    }
  });
}

__global__ __launch_bounds__(SA_ROW) void sample_draw_kernel(SampleDesc d) {
  __shared__ SampleShared sh;
  __shared__ double powers[256];
  const int row = blockIdx.x, tid = threadIdx.x;
  const Filters f = filters_of(d, row);
  const float u = uniform_of(d, row);
  fill_powers(powers);
  const float* max_of = d.block_max + (int64_t)row * d.blocks;
  const u64* mass_of = d.block_mass + (int64_t)row * d.blocks;
  float top = SA_NEG_INF, least = -SA_NEG_INF;
  for (int b = tid; b < d.blocks; b += SA_ROW) top = fmaxf(top, max_of[b]);
  block_extremes<SA_ROW>(top, least, sh.extremes);
  if (top == SA_NEG_INF) {
    if (tid == 0) no_token(d, row);
    return;
  }
  if (f.greedy) {
    int arg = 0x7fffffff;
    for (int b = tid; b < d.blocks; b += SA_ROW)
      if (max_of[b] == top) arg = min(arg, d.block_arg[(int64_t)row * d.blocks + b]);
    arg = block_least<SA_ROW>(arg, sh.least);
    if (tid == 0) sure_token(d, row, arg);
    return;
  }
  const bool infinite = top == -SA_NEG_INF;
  const Row r(f, top, top, d.shift, powers);
  const double unit = ldexp(1., -SA_BLOCK_SHIFT);
  draw<true>(
      d, row, u, r, infinite, ~0ull,
      [&](int b) {
        const float m = infinite ? tame(max_of[b]) : max_of[b];
        return (u64)__builtin_rint((double)mass_of[b] * r.scaled(m) * unit);
      },
      [&](int b) { return Row(f, max_of[b], max_of[b], SA_BLOCK_SHIFT, powers); }, sh);
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
  // Workgroups for the whole card, four to a CU, a block at least to each of
  // their waves; 64 stretches at most, as each of the next kernel's waves looks
  // into the histograms of all of them.
  const int waves = SA_SPREAD / 64;
  const int want = rows ? (int)std::min<int64_t>(64, std::max<int64_t>(1, 1024 / rows)) : 1;
  d.per_cut = ((d.blocks + want - 1) / want + waves - 1) / waves * waves;
  d.cuts = (d.blocks + d.per_cut - 1) / d.per_cut;
  d.shift = std::min(51, 62 - log2_up(vocab));
  return RTENHIP_OK;
}

// Blocks that each wave of a row's workgroup would hold.
static int held_blocks(const SampleDesc& d) { return (d.blocks + SA_ROW / 64 - 1) / (SA_ROW / 64); }

// Lays the workspace out from `base`; its size, which does not depend on the
// filters.
static size_t sample_layout(SampleDesc& d, char* base) {
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    char* p = base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t rows = (size_t)d.rows;
  d.block_mass = (u64*)take(rows * d.blocks * 8);
  d.block_max = (float*)take(rows * d.blocks * 4);
  d.block_arg = (int*)take(rows * d.blocks * 4);
  if (held_blocks(d) > 2) {
    d.cut_max = (float*)take(rows * d.cuts * 4);
    d.cut_min = (float*)take(rows * d.cuts * 4);
    d.cut_arg = (int*)take(rows * d.cuts * 4);
    d.hist = take(rows * d.cuts * SA_HIST_BYTES);
    d.list = (u64*)take(rows * SA_CAP * 8);
    d.listed = (uint32_t*)take(rows * 4);
    d.plans = (RowPlan*)take(rows * sizeof(RowPlan));
  }
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
  // Top-p of a small top-k set is decided among that set's gathered tokens.
  d.counts = k;
  d.masses = p && (sampling->top_ks || !k || sampling->top_k > SA_FEW);
  DeviceScope on(reinterpret_cast<Ctx*>(ctx)->device);
  if (on.status) return on.status;
  hipStream_t s = stream_of(ctx);
  const dim3 grid((unsigned)d.rows * (unsigned)d.cuts), rows((unsigned)d.rows), spread(SA_SPREAD), whole(SA_ROW);
  const bool none = greedy || (!k && !p);
  const bool plain = !greedy && none && !sampling->min_ps && !(sampling->min_p > 0.f);
  // One or two blocks to a wave are held (64 rows of 32,768, then of 32,769 by
  // the cut kernels: top-p 21 and 29 us, top-50 11 and 25), but two not without
  // a filter, where the cut kernels read once and take two launches (13 and 10
  // us; one row 12 and 8).
  const int held = held_blocks(d);
  if (held == 1) {
    hipLaunchKernelGGL((sample_row_kernel<1>), rows, whole, 0, s, d);
  } else if (held == 2 && !plain) {
    hipLaunchKernelGGL((sample_row_kernel<2>), rows, whole, 0, s, d);
  } else if (plain || greedy) {
    hipLaunchKernelGGL(sample_block_kernel, grid, spread, 0, s, d);
    hipLaunchKernelGGL(sample_draw_kernel, rows, whole, 0, s, d);
  } else {
    if (none) d.hist = nullptr;
    hipLaunchKernelGGL(sample_top_kernel, grid, spread, 0, s, d);
    if (d.hist) hipLaunchKernelGGL(sample_hist_kernel, grid, spread, 0, s, d);
    hipLaunchKernelGGL(sample_gather_kernel, grid, spread, 0, s, d);
    hipLaunchKernelGGL(sample_pick_kernel, rows, whole, 0, s, d);
  }
  RTENHIP_LAUNCH_CHECK();
  return RTENHIP_OK;
}
