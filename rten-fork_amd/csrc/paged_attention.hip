// Attention of new tokens over a paged cache (rtenhip_paged_attention_f32).
//
//   out = sum_j softmax_j(scale q . k_j) v_j   over the tokens j that q sees,
//
// one pass over the keys and values with a running maximum m and sum l of the
// softmax (base 2: q is multiplied by scale * log2 e once).  The query heads
// that share a cache head are rows of one tile, so keys and values are read
// once for all of them.
//
// A sequence with at most 16 rows (new tokens x heads of a group) runs in
// decode_kernel, where the cache streams from memory straight into the
// registers of the matrix instructions; the others run in chunk_kernel, up to
// 256 rows a workgroup, where tiles of keys and values are shared through LDS.
// Lengths live on the device, so each workgroup finds its own piece of work
// (plan): the visible keys of all sequences, counted in tiles of 64, are
// divided into stretches of about equal length, one to a workgroup.  Where a
// tile of rows has several stretches, merge_kernel joins their results.
#include "decoder.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rtenhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int PA_THREADS = 256;
constexpr int PA_UNIT = 64;    // keys of a tile
constexpr int PA_SMALL = 16;   // rows of a decode tile
constexpr float NEG_INF = -__builtin_huge_valf();

// What merge_kernel has to know of a stretch.
struct Part {
  int slot, part, parts, stride;  // stretches of a tile are `stride` slots apart
  int token0, row0, rows, head;
};

struct PagedDesc {
  const float* q;
  int64_t q_t, q_h;
  float* out;
  int64_t o_t, o_h;
  CacheView c;
  SeqView s;
  FastDiv group_div;
  int group, window, sinks;
  float scale_log2e;
  float minus1;  // -1, where the compiler must not know it (see split16)
  // Workspace: the stretches of the decode grid, then those of the chunk grid.
  int grid_small, grid_big, slots_small, slots_big;
  int target_small, target_big, rows_big;
  int* slots;        // stretches to join: [decode, chunk]
  Part* part_small;  // [slots]
  Part* part_big;
  float* o_small;  // [slots][PA_SMALL][dim] normalised results
  float* o_big;    // [slots][rows of a chunk tile][dim]
  float2* ml_small;  // [slots][PA_SMALL] (m, l)
  float2* ml_big;
};

// ---- plan ------------------------------------------------------------------------

// The tiles of TN keys that positions p0 .. p1 see: those of the sinks from 0
// on and then those from lo on.
struct Span {
  int sink_tiles, lo_tile, tiles;
  int lo, end;  // keys in [0, sinks) and [lo, end) are seen by some row
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : i - sink_tiles + lo_tile; }
};

template <int TN>
__device__ __forceinline__ Span span_of(const PagedDesc& d, int kv_len, int p0, int p1) {
  Span v;
  // (A tile's last key stays below 2^31.)
  const int64_t room = min((int64_t)d.s.max_pages * d.c.page_size, (int64_t)0x7fffff00);
  int end = kv_len < room ? kv_len : (int)room;
  end = min(end, p1 + 1);
  v.end = max(end, 0);
  v.lo = 0;
  v.sink_tiles = 0;
  if (d.window) {
    const int64_t lo = (int64_t)p0 - d.window + 1;
    v.lo = lo < 0 ? 0 : (int)lo;
    v.lo_tile = v.lo / TN;
    v.sink_tiles = min((min(d.sinks, v.end) + TN - 1) / TN, v.lo_tile);
  }
  v.lo_tile = v.lo / TN;
  v.tiles = v.sink_tiles + max(0, (v.end + TN - 1) / TN - v.lo_tile);
  return v;
}

// The last key that position `pos` sees as a sink only, -1 without a window.
__device__ __forceinline__ int sinks_only(const PagedDesc& d, int pos) {
  return d.window ? max(-1, (int)max((int64_t)pos - d.window, (int64_t)-1)) : -1;
}

struct Work {
  int seq, start, q_len, kv_len;
  int tile, head, part, parts, slot;
};

struct SeqWork {
  int start, q_len, kv_len, tiles, units;  // tiles of rows, tiles of keys
};

template <bool BIG, int ROWS>
__device__ __forceinline__ SeqWork seq_work(const PagedDesc& d, int s) {
  SeqWork w;
  w.start = seq_start(d.s, s);
  w.q_len = max(0, seq_start(d.s, s + 1) - w.start);
  w.kv_len = max(0, d.s.kv_lens[s]);
  const int64_t rows = (int64_t)w.q_len * d.group;
  w.units = 0;
  if (BIG)
    w.tiles = rows > PA_SMALL ? (int)((rows + ROWS - 1) / ROWS) : 0;
  else
    w.tiles = rows > 0 && rows <= PA_SMALL;
  if (w.tiles) w.units = max(1, span_of<PA_UNIT>(d, w.kv_len, w.kv_len - w.q_len, w.kv_len - 1).tiles);
  return w;
}

struct PlanShared {
  int64_t units[8];  // of each wave
  int items[8], slots[8];
  Work work;
};

// The stretches that a tile of rows over `units` tiles of keys is cut into:
// its share of the target, to the nearest.
__device__ __forceinline__ int parts_of(int units, float ratio) {
  return max(1, min(units, (int)__fmaf_rn((float)units, ratio, 0.5f)));
}

// The piece of work of workgroup `block`: false if there is none.  Every
// workgroup counts for itself (thread i the sequences i * each ..), which
// costs no launch and no order between workgroups.
template <bool BIG, int THREADS, int ROWS>
__device__ bool plan(const PagedDesc& d, int block, PlanShared& sh, Work& out) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int each = (d.s.n + THREADS - 1) / THREADS;
  const int s0 = tid * each, s1 = min(d.s.n, s0 + each);
  const int heads = d.c.heads;
  // (The first one's is kept: mostly there is no other, and its lengths take a
  // round trip to memory each time.)
  SeqWork first{};
  if (s0 < s1) first = seq_work<BIG, ROWS>(d, s0);
  const auto work_of = [&](int s) { return s == s0 ? first : seq_work<BIG, ROWS>(d, s); };
  int64_t units = 0;
  for (int s = s0; s < s1; s++) {
    const SeqWork w = work_of(s);
    units += (int64_t)w.tiles * w.units;
  }
  units = (int64_t)wave_sum((u64)units);
  if (lane == 0) sh.units[wave] = units;
  if (tid == 0) sh.work.seq = -1;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) total += sh.units[i] * heads;
  const float ratio = (float)(BIG ? d.target_big : d.target_small) / (float)total;
  int items = 0, slots = 0;
  for (int s = s0; s < s1; s++) {
    const SeqWork w = work_of(s);
    const int parts = parts_of(w.units, ratio);
    const int n = w.tiles * heads * parts;
    items += n;
    slots += parts > 1 ? n : 0;
  }
  const int items_in = (int)wave_scan((uint32_t)items), slots_in = (int)wave_scan((uint32_t)slots);
  if (lane == 63) sh.items[wave] = items_in, sh.slots[wave] = slots_in;
  __syncthreads();
  if (block == 0 && tid == 0 && d.slots) {
    int n = 0, all = 0;
    for (int w = 0; w < THREADS / 64; w++) n += sh.slots[w], all += sh.items[w];
    // (More pieces than workgroups: q_starts do not rise, and some stretches
    // never come.  Nothing is joined then.)
    d.slots[BIG] = all > (int)gridDim.x ? 0 : min(n, BIG ? d.slots_big : d.slots_small);
  }
  int at = items_in - items, slot = slots_in - slots;
  for (int w = 0; w < wave; w++) at += sh.items[w], slot += sh.slots[w];
  if (block >= at && block < at + items) {
    for (int s = s0; s < s1; s++) {
      const SeqWork w = work_of(s);
      const int parts = parts_of(w.units, ratio);
      const int n = w.tiles * heads * parts;
      if (block < at + n) {
        int i = block - at;
        Work r;
        r.seq = s, r.start = w.start, r.q_len = w.q_len, r.kv_len = w.kv_len;
        r.slot = parts > 1 ? slot + i : -1;
        r.head = i % heads;
        i /= heads;
        r.part = i % parts;
        r.parts = parts;
        r.tile = w.tiles - 1 - i / parts;  // the last rows see the most keys: first
        sh.work = r;
        break;
      }
      at += n;
      slot += parts > 1 ? n : 0;
    }
  }
  __syncthreads();
  // (In scalar registers: everything that follows from it is the same for all
  // lanes, loops and addresses among it.)
  static_assert(sizeof(Work) % 4 == 0, "copied word by word");
  const int* from = (const int*)&sh.work;
  int* to = (int*)&out;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(Work) / 4); i++) to[i] = __builtin_amdgcn_readfirstlane(from[i]);
  return out.seq >= 0;
}

// ---- small pieces ------------------------------------------------------------------

__device__ __forceinline__ float half_max(float x) {  // with lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float quarter_max(float x) {  // over lanes ^ 16, ^ 32
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarter_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true));
}
// The largest of numbers of which none is negative (their bits are in the same
// order): over every 8 lanes, and from those over the wave.
__device__ __forceinline__ uint32_t eighth_max(float y) {
  uint32_t x = __float_as_uint(y);
  x = max_dpp<0xB1>(x);         // lane ^ 1
  x = max_dpp<0x4E>(x);         // lane ^ 2
  return max_dpp<0x141>(x);     // mirrored in its 8
}
__device__ __forceinline__ uint32_t wave_max_of_eighths(uint32_t x) {
  x = max_dpp<0x140>(x);  // mirrored in its 16
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(r[0], r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(s[0], s[1]);
}
// The smallest, likewise.
__device__ __forceinline__ uint32_t wave_min_of_eighths(uint32_t x) {
  x = min(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = min(r[0], r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return min(s[0], s[1]);
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
  x = min(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
  x = min(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
  x = min(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));
  return wave_min_of_eighths(x);
}
// The largest, over every 32 lanes, of the lanes' two 16-bit numbers each.
__device__ __forceinline__ u16x2 half_max16(u16x2 x) {
  const auto step = [](u16x2 a, int b) { return __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, b)); };
  x = step(x, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, true));
  x = step(x, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, true));
  x = step(x, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x141, 0xF, 0xF, true));
  x = step(x, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x140, 0xF, 0xF, true));
  const uint32_t y = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return step(__builtin_bit_cast(u16x2, (uint32_t)r[0]), (int)r[1]);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The power of two that brings a largest magnitude `big` to [2^13, 2^14), as
// an exponent; what is not finite or very small counts as the nearest that is
// in range, zero as 2^-100.
__device__ __forceinline__ int exponent_for(float big) {
  int e = (int)((__float_as_uint(big) >> 23) & 255) - 127;
  e = e > 127 ? 127 : e < -100 ? -100 : e;
  return 13 - e;
}
__device__ __forceinline__ float pow2(int e) {  // e brought into the normal range
  e = e < -126 ? -126 : e > 127 ? 127 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// x, of which the compiler does not know where it comes from (no instruction).
template <typename T>
__device__ __forceinline__ T opaque(T x) {
  static_assert(sizeof(T) == 4, "one register");
  asm("" : "+v"(x));
  return x;
}

// x = hi + lo in f16: 22 bits of x where |x| is within 2^14 and above 2^-3,
// an absolute error of 2^-25 below that.  lo is x - hi exactly, by one mixed
// fma that reads hi from its half of the register, before its own rounding:
// the -1 has to be a register for that, and hi not be seen to be a conversion,
// which would be repeated for each half.
__device__ __forceinline__ void split16(float a, float b, float minus1, f16x2& hi, f16x2& lo) {
  hi = opaque((f16x2){(_Float16)a, (_Float16)b});
  lo = (f16x2){(_Float16)__builtin_fmaf((float)hi[0], minus1, a), (_Float16)__builtin_fmaf((float)hi[1], minus1, b)};
}
// The same of a f and b g, f and g powers of two.
__device__ __forceinline__ void split16(float a, float b, float f, float g, f16x2& hi, f16x2& lo) {
  hi = opaque((f16x2){(_Float16)(a * f), (_Float16)(b * g)});
  lo = (f16x2){(_Float16)__builtin_fmaf(a, f, -(float)hi[0]), (_Float16)__builtin_fmaf(b, g, -(float)hi[1])};
}

template <int TYPE>
struct CacheType {
  static constexpr int size = TYPE == RTENHIP_CACHE_F32 ? 4 : 2;
};

// ---- decode --------------------------------------------------------------------------

// Sixteen rows at most; each of the 4 waves takes 16 keys of every tile of 64
// and keeps its own m, l and result, joined through LDS at the end.
//  - S^T = K Q^T: lane (i, g) (i < 16, g < 4) loads parts of key i's row as
//    they lie and feeds them to the matrix instruction as they are: which of
//    the dimensions a step multiplies does not matter as long as Q's register
//    holds the same ones.  The lane then has the scores of row i for the keys
//    4g .. 4g + 3.
//  - O^T = V^T P^T: those four are the P operand as they are, and the lane
//    loads the values of keys 4g .. 4g + 3 for DP / 16 neighbouring
//    dimensions, so nothing moves between lanes.
// An f32 cache uses the f32 instructions, f16 splits q and p into two f16
// terms (exact products, 22 bits of q and p), bf16 into three bf16 terms.
// Bound by the cache's bytes: DEPTH tiles are on their way in registers while
// one is worked on.  64 ragged sequences of 60 to 6000 keys (f16, 8 heads of
// 128, 0.80 GB): 160 us, 5.0 TB/s; 131,072 keys of one sequence (f32, 1.07 GB):
// 188 us with the join, 5.7 TB/s; 32 windows of 4096 (bf16, 8 heads of 64, 0.27
// GB): 64 us, 4.2 TB/s.  A copy of 4 GiB runs at 4.7.  The matrix instructions
// are busy for 9, 27 and 11 % of the time.
template <int DP, int TYPE>
struct DecodeTile {
  static constexpr int DPL = DP / 16;                                // value dimensions of a lane
  static constexpr int KV = DP * CacheType<TYPE>::size / 64;         // 16-byte loads of keys
  static constexpr int VW = DPL * CacheType<TYPE>::size / 4;         // 32-bit words of values, per key
  // Waves on a SIMD, and tiles in flight in each.  (Two tiles in flight against
  // one on 64 sequences of up to 6000 keys, f16, head_dim 128: 177 against 182
  // us; of f32 rows, twice as long, one is enough: 188 against 208 us over
  // 131,072 keys, where two leave no registers.  Windows of bf16 rows of 64:
  // 64 us with 3 waves, 63 with 2 and 67 with 4; ragged sequences of them 104,
  // 110 and 110.  f32 rows of 256, 64 ragged sequences: 684 us with one wave,
  // 1206 with two, which spill; 16-bit rows would take two, f16 308 us for 341.)
  static constexpr int WAVES = DP == 64 ? 3 : DP == 128 ? 2 : 1;
  static constexpr int DEPTH = DP == 64 || (DP == 128 && TYPE != RTENHIP_CACHE_F32) ? 2 : 1;
  static constexpr int QW = TYPE == RTENHIP_CACHE_F32 ? DP / 4 : TYPE == RTENHIP_CACHE_F16 ? DP / 4 : 3 * DP / 8;
};

// Rows are loaded whether there is a key or not (then the cache's first row,
// which there always is), and what must not count is cleared when it is used: a
// load under a condition would be waited for where the paths meet.
// Past head_dim the row's last 16 bytes are read again: q is zero there, and
// those results are not stored.
template <int DP, int TYPE>
__device__ __forceinline__ void load_keys(const char* row, int g, int dim, u32x4* k) {
  constexpr int KV = DecodeTile<DP, TYPE>::KV, size = CacheType<TYPE>::size, per = 16 / size;
#pragma unroll
  for (int j = 0; j < KV; j++) k[j] = *(const u32x4*)(row + min((4 * j + g) * per, dim - per) * size);
}

// The same, and the words of load_words, from a row at a scalar address that all
// lanes share, with each lane's own offset: nothing is left to add.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t from_here(const char* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, -1, 0x00020000);
}
template <int WORDS>
__device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t base, const uint32_t* lane, uint32_t row, uint32_t* v) {
  if constexpr (WORDS == 1) {
    v[0] = __builtin_amdgcn_raw_buffer_load_b32(base, lane[0], row, 0);
  } else if constexpr (WORDS == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(base, lane[0], row, 0);
    v[0] = x[0], v[1] = x[1];
  } else {
#pragma unroll
    for (int c = 0; c < WORDS; c += 4) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b128(base, lane[c / 4], row, 0);
#pragma unroll
      for (int e = 0; e < 4; e++) v[c + e] = x[e];
    }
  }
}

// WORDS words at byte `at` of a row of `bytes` bytes, its last ones where there
// are fewer.
template <int WORDS>
__device__ __forceinline__ void load_words(const char* row, int at, int bytes, uint32_t* v) {
  if constexpr (WORDS == 1) {
    v[0] = *(const uint32_t*)(row + min(at, bytes - 4));
  } else if constexpr (WORDS == 2) {
    const u32x2 x = *(const u32x2*)(row + min(at, bytes - 8));
    v[0] = x[0], v[1] = x[1];
  } else {
#pragma unroll
    for (int c = 0; c < WORDS; c += 4) {
      const u32x4 x = *(const u32x4*)(row + min(at + 4 * c, bytes - 16));
#pragma unroll
      for (int e = 0; e < 4; e++) v[c + e] = x[e];
    }
  }
}

// The words of a key's or value's row with what is not finite set to zero;
// true if there was any.
template <int TYPE>
__device__ __forceinline__ bool clean(uint32_t& w) {
  if constexpr (TYPE == RTENHIP_CACHE_F32) {
    const bool bad = (w & 0x7f800000u) == 0x7f800000u;
    if (bad) w = 0;
    return bad;
  } else {
    constexpr uint32_t e = TYPE == RTENHIP_CACHE_F16 ? 0x7c00u : 0x7f80u;
    const bool lo = (w & e) == e, hi = (w & (e << 16)) == (e << 16);
    if (lo) w &= 0xffff0000u;
    if (hi) w &= 0x0000ffffu;
    return lo || hi;
  }
}

// ALIGNED: no page ends inside a wave's 16 keys (decode_aligned), so they have
// one page and their rows' distances fit 32 bits: a tile's addresses are two
// scalars, and registers that stay.  Otherwise each lane finds its key's rows and the
// values' come from the lanes that have them.
template <int DP, int TYPE, bool ALIGNED>
__global__ __launch_bounds__(PA_THREADS, (DecodeTile<DP, TYPE>::WAVES)) void decode_kernel(PagedDesc d) {
  using T = DecodeTile<DP, TYPE>;
  constexpr int DPL = T::DPL, KV = T::KV, VW = T::VW, DEPTH = T::DEPTH, size = CacheType<TYPE>::size;
  __shared__ PlanShared plan_sh;
  __shared__ float o_sh[4][PA_SMALL][DP];
  __shared__ float m_sh[4][PA_SMALL], l_sh[4][PA_SMALL];
  Work w;
  if (!plan<false, PA_THREADS, PA_SMALL>(d, blockIdx.x, plan_sh, w) || w.slot >= d.slots_small) return;
  if (threadIdx.x == 0 && w.slot >= 0)
    d.part_small[w.slot] = Part{w.slot, w.part, w.parts, d.c.heads, w.start, 0, w.q_len * d.group, w.head};
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int i = lane & 15, g = lane >> 4;
  const int dim = d.c.dim, rows = w.q_len * d.group;
  const int token = fdiv(i, d.group_div), sub = i - token * d.group;
  const bool row_ok = i < rows;
  const int pos = row_ok ? w.kv_len - w.q_len + token : -1;
  const int below = sinks_only(d, pos);

  // Q, times scale log2 e, as the matrix instructions take it.
  uint32_t qw[T::QW];
  float q_back = 1.f;  // what the scores are multiplied by
  {
    const float* q = d.q + (int64_t)(w.start + token) * d.q_t + (int64_t)(w.head * d.group + sub) * d.q_h;
    constexpr int PER = 16 / size;
    float x[KV][PER];
#pragma unroll
    for (int j = 0; j < KV; j++) {
      const int at = (4 * j + g) * PER;
      const bool ok = row_ok && at < dim;
#pragma unroll
      for (int e = 0; e < PER; e += 4) {
        const float4 y = ok ? *(const float4*)(q + at + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[j][e] = y.x * d.scale_log2e, x[j][e + 1] = y.y * d.scale_log2e;
        x[j][e + 2] = y.z * d.scale_log2e, x[j][e + 3] = y.w * d.scale_log2e;
      }
    }
    if constexpr (TYPE == RTENHIP_CACHE_F32) {
#pragma unroll
      for (int j = 0; j < KV; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) qw[4 * j + e] = __float_as_uint(x[j][e]);
    } else if constexpr (TYPE == RTENHIP_CACHE_F16) {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < KV; j++)
#pragma unroll
        for (int e = 0; e < PER; e++) big = fmaxf(big, fabsf(x[j][e]));
      const int up = exponent_for(quarter_max(big));
      const float f = pow2(up);
      q_back = pow2(-up);
#pragma unroll
      for (int j = 0; j < KV; j++)
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
          f16x2 hi, lo;
          split16(x[j][e] * f, x[j][e + 1] * f, d.minus1, hi, lo);
          qw[4 * j + e / 2] = __builtin_bit_cast(uint32_t, hi);
          qw[DP / 8 + 4 * j + e / 2] = __builtin_bit_cast(uint32_t, lo);
        }
    } else {
#pragma unroll
      for (int j = 0; j < KV; j++)
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
          float a = x[j][e], b = x[j][e + 1];
#pragma unroll
          for (int t = 0; t < 3; t++) {
            const __bf16 ha = (__bf16)a, hb = (__bf16)b;
            qw[t * DP / 8 + 4 * j + e / 2] = (uint32_t)__builtin_bit_cast(uint16_t, ha) |
                                             (uint32_t)__builtin_bit_cast(uint16_t, hb) << 16;
            a -= (float)ha, b -= (float)hb;
          }
        }
    }
  }

  const Span span = span_of<PA_UNIT>(d, w.kv_len, w.kv_len - w.q_len, w.kv_len - 1);
  const int u0 = (int)((int64_t)span.tiles * w.part / w.parts), u1 = (int)((int64_t)span.tiles * (w.part + 1) / w.parts);
  const int* table = d.s.table + (int64_t)w.seq * d.s.table_stride;
  const char* kc = d.c.k + (int64_t)w.head * d.c.k_head * size;
  const char* vc = d.c.v + (int64_t)w.head * d.c.v_head * size;

  const int pos_first = w.kv_len - w.q_len, below_last = sinks_only(d, w.kv_len - 1);

  // Key 0 of the wave's 16 in tile u, and whether some row sees a key.
  auto key_of = [&](int u) { return span.tile(min(u, u1 - 1)) * PA_UNIT + 16 * wave; };
  auto seen_key = [&](int key) { return (key < span.end) & ((key >= span.lo) | (key < d.sinks)); };
  struct Place {
    int page, slot;
  };
  auto page_at = [&](int u) {
    const int key = key_of(u) + (ALIGNED ? 0 : i), at = fdiv(key, d.c.page_div);
    return Place{u < u1 && key < span.end && at < d.s.max_pages ? table[at] : -1, key - at * d.c.page_size};
  };
  // ALIGNED: a lane's way from its wave's first row, in bytes.
  constexpr int VL = VW < 4 ? 1 : VW / 4;
  uint32_t k_lane[KV], v_lane[VL];
  if constexpr (ALIGNED) {
    constexpr int per = 16 / size, last = VW < 4 ? VW * 4 : 16;
#pragma unroll
    for (int j = 0; j < KV; j++) k_lane[j] = (uint32_t)(i * d.c.k_slot + min((4 * j + g) * per, dim - per)) * size;
#pragma unroll
    for (int c = 0; c < VL; c++)
      v_lane[c] = (uint32_t)(4 * g * d.c.v_slot * size + min(i * DPL * size + 16 * c, dim * size - last));
  }

  float m, l;
  f32x4 o[DPL];
  bool poison;
  auto pass = [&](bool careful) __attribute__((always_inline)) {
    m = NEG_INF, l = 0.f;
    poison = false;
#pragma unroll
    for (int e = 0; e < DPL; e++) o[e] = (f32x4){0, 0, 0, 0};
    // Tile u is loaded into stage (u - u0) % DEPTH; its page was asked for two
    // loads before.
    u32x4 k[DEPTH][KV];
    uint32_t v[DEPTH][4][VW];
    uint32_t here[DEPTH];  // the wave's keys that there are, the lane's four from bit 4 g on
    Place next = page_at(u0), after = page_at(u0 + 1);
    auto fetch = [&](int u, int stage) __attribute__((always_inline)) {
      const int page = ALIGNED ? __builtin_amdgcn_readfirstlane(next.page) : next.page;
      const bool ok = page_ok(d.c, page);
      if constexpr (ALIGNED) {
        const uint32_t p = ok ? page : 0, slot = ok ? next.slot : 0;
        const uint32_t k_slot = (uint32_t)d.c.k_slot * size, v_slot = (uint32_t)d.c.v_slot * size;
        const auto kr = from_here(kc + ((uint64_t)p * (uint32_t)(d.c.k_page * size) + slot * k_slot));
        const auto vr = from_here(vc + ((uint64_t)p * (uint32_t)(d.c.v_page * size) + slot * v_slot));
#pragma unroll
        for (int j = 0; j < KV; j++) load_words<4>(kr, &k_lane[j], 0, (uint32_t*)&k[stage][j]);
#pragma unroll
        for (int r = 0; r < 4; r++) load_words<VW>(vr, v_lane, r * v_slot, v[stage][r]);
        here[stage] = ok ? 0xffff : 0;
      } else {
        const int64_t k_row = ok ? (page * d.c.k_page + next.slot * d.c.k_slot) * size : 0;
        const int64_t v_row = ok ? (page * d.c.v_page + next.slot * d.c.v_slot) * size : 0;
        load_keys<DP, TYPE>(kc + k_row, g, dim, k[stage]);
#pragma unroll
        for (int r = 0; r < 4; r++)
          load_words<VW>(vc + __shfl((long long)v_row, 4 * g + r), i * DPL * size, dim * size, v[stage][r]);
        here[stage] = (uint32_t)__ballot(ok) & 0xffff;
      }
      next = after;
      after = page_at(u + 2);
    };
    auto work = [&](int u, const u32x4* k, uint32_t (*v)[VW], uint32_t here) __attribute__((always_inline)) {
      const int key = key_of(u), base = key + 4 * g;
      // All 16 keys are seen by all rows; by some row.
      const bool some = here == 0xffff && key + 15 < span.end && (key >= span.lo || key + 15 < d.sinks);
      const bool all = some && key + 15 <= pos_first && (key > below_last || key + 15 < d.sinks);
      f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KV; j++) {
        if constexpr (TYPE == RTENHIP_CACHE_F32) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[j][e]), __uint_as_float(qw[4 * j + e]), s0, 0,
                                                      0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[j][e + 1]), __uint_as_float(qw[4 * j + e + 1]),
                                                      s1, 0, 0, 0);
          }
        } else {
          const u32x4 a = k[j];
          const auto part = [&](int t) {
            return (u32x4){qw[t * DP / 8 + 4 * j], qw[t * DP / 8 + 4 * j + 1], qw[t * DP / 8 + 4 * j + 2],
                           qw[t * DP / 8 + 4 * j + 3]};
          };
          if constexpr (TYPE == RTENHIP_CACHE_F16) {
            const f16x8 x = __builtin_bit_cast(f16x8, a);
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(f16x8, part(0)), s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(f16x8, part(1)), s1, 0, 0, 0);
          } else {
            const bf16x8 x = __builtin_bit_cast(bf16x8, a);
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, part(0)), s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, part(1)), s1, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, part(2)), s1, 0, 0, 0);
          }
        }
      }
      float p[4];
      uint32_t seen = 15;  // the lane's keys that its row sees
#pragma unroll
      for (int r = 0; r < 4; r++) p[r] = (s0[r] + s1[r]) * q_back;
      if (!all) {
        seen = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int at = base + r;
          const bool ok = (here >> (4 * g + r) & 1) & seen_key(at) & (at <= pos) & ((at > below) | (at < d.sinks));
          seen |= (uint32_t)ok << r;
          p[r] = ok ? p[r] : NEG_INF;
        }
      }
      const float m_new = fmaxf(m, quarter_max(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]))));
      const float ref = m_new == NEG_INF ? 0.f : m_new;
      if (__any(m_new > m)) {
        const float fade = __builtin_amdgcn_exp2f(m - ref);
        m = m_new;
        l *= fade;
#pragma unroll
        for (int e = 0; e < DPL; e++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[e][r] *= fade;
      }
      // f16 terms of p have the most bits where the largest p is 2^14; the
      // factor is in l too.
      constexpr float UP = TYPE == RTENHIP_CACHE_F16 ? 14.f : 0.f;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[r] = __builtin_amdgcn_exp2f(UP == 0.f ? p[r] - ref : (p[r] - ref) + UP);
        l += p[r];
      }
      if (!some) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool ok = (here >> (4 * g + r) & 1) & seen_key(base + r);
#pragma unroll
          for (int c = 0; c < VW; c++) v[r][c] = ok ? v[r][c] : 0;
        }
      }
      if (careful) {
        // A value that is not finite must not meet the zero weight of a row
        // that does not see it; the rows that do see it end as NaN.
#pragma unroll
        for (int r = 0; r < 4; r++) {
          bool bad = false;
#pragma unroll
          for (int c = 0; c < VW; c++) bad |= clean<TYPE>(v[r][c]);
          const bool key_bad = (__ballot(bad) >> (16 * g)) & 0xffff;
          poison |= key_bad & (seen >> r & 1);
        }
      }
      if constexpr (TYPE == RTENHIP_CACHE_F32) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int e = 0; e < DPL; e++)
            o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][e]), p[r], o[e], 0, 0, 0);
      } else {
        // Four keys' values of a dimension side by side.
        const auto column = [&](int e) {
          const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
          return (u32x2){__builtin_amdgcn_perm(v[1][e / 2], v[0][e / 2], sel),
                         __builtin_amdgcn_perm(v[3][e / 2], v[2][e / 2], sel)};
        };
        if constexpr (TYPE == RTENHIP_CACHE_F16) {
          f16x2 h0, l0, h1, l1;
          split16(p[0], p[1], d.minus1, h0, l0);
          split16(p[2], p[3], d.minus1, h1, l1);
          const f16x4 hi = {h0[0], h0[1], h1[0], h1[1]}, lo = {l0[0], l0[1], l1[0], l1[1]};
#pragma unroll
          for (int e = 0; e < DPL; e++) {
            const f16x4 a = __builtin_bit_cast(f16x4, column(e));
            o[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, hi, o[e], 0, 0, 0);
            o[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(a, lo, o[e], 0, 0, 0);
          }
        } else {
          s16x4 terms[3];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            float x = p[r];
#pragma unroll
            for (int t = 0; t < 3; t++) {
              const __bf16 h = (__bf16)x;
              terms[t][r] = __builtin_bit_cast(short, h);
              x -= (float)h;
            }
          }
#pragma unroll
          for (int e = 0; e < DPL; e++) {
            const s16x4 a = __builtin_bit_cast(s16x4, column(e));
#pragma unroll
            for (int t = 0; t < 3; t++) o[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, terms[t], o[e], 0, 0, 0);
          }
        }
      }
    };
#pragma unroll
    for (int s = 0; s < DEPTH; s++) fetch(u0 + s, s);
    for (int u = u0; u < u1; u += DEPTH) {
#pragma unroll
      for (int s = 0; s < DEPTH; s++) {
        if (u + s < u1) work(u + s, k[s], v[s], here[s]);
        fetch(u + s + DEPTH, s);
      }
    }
    l = quarter_sum(l);
  };
  // A result that is not finite may come from a value that its row does not
  // see: once more, with care.
  for (int k = 0; k < 2; k++) {
    pass(k);
    bool bad = !finite(l);
#pragma unroll
    for (int e = 0; e < DPL; e++)
#pragma unroll
      for (int r = 0; r < 4; r++) bad |= !finite(o[e][r]);
    if (!__any(bad)) break;
  }
  if (quarter_max(poison ? 1.f : 0.f) > 0.f) l = __builtin_nanf("");
  if (g == 0) m_sh[wave][i] = m, l_sh[wave][i] = l;
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int e = 0; e < DPL; e += 4)
      *(f32x4*)&o_sh[wave][i][DPL * (4 * g + r) + e] = (f32x4){o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
  __syncthreads();
  const int quads = dim / 4;
  for (int at = tid; at < rows * quads; at += PA_THREADS) {
    const int row = at / quads, c = (at - row * quads) * 4;
    const float m_all = fmaxf(fmaxf(m_sh[0][row], m_sh[1][row]), fmaxf(m_sh[2][row], m_sh[3][row]));
    const float ref = m_all == NEG_INF ? 0.f : m_all;
    f32x4 sum = {0, 0, 0, 0};
    float l_all = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float f = __builtin_amdgcn_exp2f(m_sh[k][row] - ref);
      l_all = __fmaf_rn(l_sh[k][row], f, l_all);
      const f32x4 x = *(const f32x4*)&o_sh[k][row][c];
#pragma unroll
      for (int e = 0; e < 4; e++) sum[e] = __fmaf_rn(x[e], f, sum[e]);
    }
    const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] *= inv;
    if (w.slot < 0) {
      const int tok = row / d.group;
      *(f32x4*)(d.out + (int64_t)(w.start + tok) * d.o_t + (int64_t)(w.head * d.group + row - tok * d.group) * d.o_h +
                c) = sum;
    } else {
      *(f32x4*)(d.o_small + ((int64_t)w.slot * PA_SMALL + row) * dim + c) = sum;
      if (c == 0) d.ml_small[(int64_t)w.slot * PA_SMALL + row] = make_float2(m_all, l_all);
    }
  }
}

// ---- chunk ---------------------------------------------------------------------------

// 256 rows (new token, head of the group) a workgroup, 32 a wave.  Tiles of
// keys and values go to LDS as f16 terms, and both products run on the f16
// matrix instructions:
//  - an f32 number x 2^e is hi + lo, each f16 (split16), and a product
//    hi hi + hi lo + lo hi, three f16 instructions against the eight times
//    longer f32 one, loses what is below 2^-22 of it; a 16-bit cache needs no
//    lo.  e is one power of two for every 8 keys and one for their values, so
//    that the largest number of either is near 2^13 and the terms are exact to
//    2^-38 of it; q has one for each row, p the factor 2^8.  Powers of two come
//    out again exactly: a score is multiplied by its keys' and its row's on
//    its way into the exponential, whose argument takes the values'.
//    Not all rows see all of 8 keys, and a loud one must not cost its
//    neighbours their bits: where the largest numbers of 8 keys, or of their
//    values, are more than 2^EVEN apart (an infinity always is), or values more
//    than 2^FALL below the loudest before them or in their tile, the stretch is
//    computed again with a power of two for each key and each value's row, and
//    the products of values of different loudness apart (careful).  Up to there
//    a row is exact to 2^-26 of its own largest number and p to 2^-23 of the
//    largest p, finer than the split's 22 bits.  (Values below 2^-93 lose bits
//    beside others above 2^53 in either pass.)
//  - S^T = K Q^T: a lane (n, h) has row n's scores for the keys
//    8 i + 4 h + j of each 32, so the softmax needs one exchange with lane
//    ^ 32, and
//  - O^T = V^T P^T takes them as they lie: LDS holds V^T with the keys of
//    every 16 in the order (h, i, j), 16 bytes for a lane's eight.
//  The maximum that p is taken against follows the largest score only when it
//  is passed by more than 2^6, which few tiles do, so the result is hardly
//  ever rescaled.
// Two LDS buffers and one barrier a tile: while tile u is multiplied, u + 1 is
// converted into the other buffer, 8 keys by each wave, and u + 2 is on its way
// into registers.  Eight waves, two to a SIMD: one of the two converts before
// it multiplies and the other after, which keeps one's conversions and
// exponentials under the other's products; at head_dim 256 a wave needs all of
// a SIMD's registers, and four waves work on tiles of 32 keys.
// Bound by the matrix instructions, and what has to be converted between them,
// at long prompts: 8192 tokens of 32 heads of 128 on an f32 cache, 550 GFLOP and
// three f16 products for each, 1.6 ms, 1.0 PFLOP/s of them (a library's f16
// product of 8192^3: 1.19; f32 instructions alone would take 3.6 ms).  Matrix
// instructions run for 49 % of the SIMDs' cycles, vector ones issue for 51 %.
// 4096 tokens on a bf16 cache 0.32 ms, on f16 0.29; 2048 tokens of 16 heads of
// 256, f32, 0.30 ms.
template <int DP, int TYPE>
struct ChunkTile {
  static constexpr int WAVES = DP == 256 ? 4 : 8, THREADS = 64 * WAVES;
  static constexpr int TN = DP == 256 ? 32 : 64;  // keys of a tile
  static constexpr int ROWS = 32 * WAVES;
  static constexpr int TERMS = TYPE == RTENHIP_CACHE_F32 ? 2 : 1;
  static constexpr int KS = DP * 2 + 16;  // bytes of a key's row in LDS, off by a bank group per row
  static constexpr int KL = DP * CacheType<TYPE>::size / 128;     // 16-byte loads of keys per thread (8 to a row)
  static constexpr int DPV = DP / 32;                             // value dimensions per thread, of 4 keys
  static constexpr int VW = DPV * CacheType<TYPE>::size / 4;      // words of values per thread and key
  static constexpr int K_BYTES = TN * KS, V_BYTES = DP * TN * 2;
  static constexpr int BUFFER = TERMS * (K_BYTES + V_BYTES);
};

// Rows of a chunk tile (what the plan counts in).
template <int DP>
constexpr int chunk_rows() {
  return ChunkTile<DP, RTENHIP_CACHE_F32>::ROWS;
}

// Where the 16 bytes of keys (h, i, j), chunk = 2 * (16 keys) + h, of a
// dimension lie: the chunks of neighbouring dimensions, and of dimensions 8
// apart, are in different banks.
template <int TN>
__device__ __forceinline__ int value_at(int dimension, int chunk) {
  if constexpr (TN == 64) return dimension * 128 + ((chunk ^ dimension ^ (dimension >> 3)) & 7) * 16;
  return dimension * 64 + ((chunk ^ (dimension >> 1) ^ (dimension >> 3)) & 3) * 16;
}
// value_at(32 b + n, chunk + h) for n < 32, even chunks and h < 2 is
// value_at(n, h) with these bits flipped and 32 b rows on.
template <int TN>
__device__ __forceinline__ constexpr int value_flip(int dimension, int chunk) {
  if (TN == 64) return ((chunk ^ (dimension >> 3)) & 7) * 16;
  return ((chunk ^ (dimension >> 1) ^ (dimension >> 3)) & 3) * 16;
}

template <int TYPE>
__device__ __forceinline__ float cache_lo(uint32_t w) {
  if constexpr (TYPE == RTENHIP_CACHE_F16) return (float)__builtin_bit_cast(f16x2, w)[0];
  return __uint_as_float(w << 16);
}
template <int TYPE>
__device__ __forceinline__ float cache_hi(uint32_t w) {
  if constexpr (TYPE == RTENHIP_CACHE_F16) return (float)__builtin_bit_cast(f16x2, w)[1];
  return __uint_as_float(w & 0xffff0000u);
}

// The largest magnitude among `top` and two words of the cache; a NaN counts as
// nothing.  (The instruction takes magnitudes as it goes; fmaxf would first
// quiet what comes from memory.)
template <int TYPE>
__device__ __forceinline__ float top_of(float top, uint32_t x, uint32_t y) {
  const auto max3 = [](float a, float b, float c) {
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(a) : "v"(a), "v"(b), "v"(c));
    return a;
  };
  if constexpr (TYPE == RTENHIP_CACHE_F32) return max3(top, __uint_as_float(x), __uint_as_float(y));
  return max3(max3(top, cache_lo<TYPE>(x), cache_hi<TYPE>(x)), cache_lo<TYPE>(y), cache_hi<TYPE>(y));
}

// What is known of a tile in LDS: the exponents of every 8 keys and of their
// values, and by bits the keys that somebody sees and those with a value that
// is not finite.
struct __attribute__((aligned(16))) TileInfo {
  int8_t k_up[8], v_up[8];
  uint64_t seen, bad;
};

// How many binades the largest numbers of 8 keys may lie apart to share an
// exponent, how many the values of a tile below the result's scale, and that
// scale's least exponent (2^27 values of 2^127 can be added, and there are 85
// binades below 1).
constexpr uint32_t EVEN = 12;
constexpr int FALL = 10, O_LEAST = -41;
constexpr int NO_VALUE = 127;  // the exponent of values that are all zero (or below 2^-133)

// x, of which the compiler does not know that it is the same in every round of
// a loop: what follows from it is formed again there, a few instructions,
// instead of being held in a register that the products' operands need.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Steps 0 .. STEPS - 1, each reading its operands from LDS (read) and then
// multiplying them (multiply): the reads are AHEAD steps before the products,
// which the compiler, short of registers, would put right behind them.
template <int STEPS, int AHEAD, typename Operands, typename Read, typename Multiply>
__device__ __forceinline__ void pipelined(Read read, Multiply multiply) {
  Operands x[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; i++) x[i] = read(i);
#pragma unroll
  for (int i = 0; i < STEPS; i++) {
    __builtin_amdgcn_sched_barrier(0);
    multiply(i, x[i % AHEAD]);
    __builtin_amdgcn_sched_barrier(0);
    if (i + AHEAD < STEPS) x[i % AHEAD] = read(i + AHEAD);
  }
}

template <int DP, int TYPE>
__global__ __launch_bounds__((ChunkTile<DP, TYPE>::THREADS), DP == 256 ? 1 : 2) void chunk_kernel(PagedDesc d) {
  using T = ChunkTile<DP, TYPE>;
  constexpr int TERMS = T::TERMS, KS = T::KS, KL = T::KL, VW = T::VW, DPV = T::DPV, TN = T::TN, WAVES = T::WAVES;
  constexpr int size = CacheType<TYPE>::size, PER = 16 / size, NB = DP / 32;
  constexpr bool SCALED = TYPE != RTENHIP_CACHE_F16;  // f16 rows go to LDS as they are
  constexpr int AHEAD = 2;  // LDS reads before their products, in steps
  struct Operands {
    f16x8 term[TERMS];
  };
  __shared__ PlanShared plan_sh;
  __shared__ __attribute__((aligned(16))) char buffer_sh[2][T::BUFFER];  // keys hi, lo, values hi, lo
  // [tile & 3], as they are read late.
  __shared__ int64_t rows_sh[4][2][TN];  // the keys' and the values' rows
  __shared__ TileInfo info_sh[4];
  // Each key's exponent and its value's, with care.
  __shared__ __attribute__((aligned(4))) int8_t key_up_sh[SCALED ? 4 : 1][TN], value_up_sh[SCALED ? 4 : 1][TN];
  __shared__ int uneven_sh;
  Work w;
  if (!plan<true, T::THREADS, T::ROWS>(d, blockIdx.x, plan_sh, w) || w.slot >= d.slots_big) return;
  const int row0 = w.tile * T::ROWS;
  const int all_rows = w.q_len * d.group;
  const int rows = min(T::ROWS, all_rows - row0);
  if (threadIdx.x == 0 && w.slot >= 0)
    d.part_big[w.slot] = Part{w.slot, w.part, w.parts, d.c.heads, w.start, row0, rows, w.head};
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int n = lane & 31, h = lane >> 5;
  const int dim = d.c.dim, first = w.kv_len - w.q_len;
  const int wave_row = row0 + wave * 32;
  const bool wave_ok = wave_row < all_rows;
  const int row = wave_row + n;
  const bool row_ok = row < all_rows;
  const int token = fdiv(row_ok ? row : 0, d.group_div), sub = row_ok ? row - token * d.group : 0;
  const int pos = row_ok ? first + token : -1;
  const int below = sinks_only(d, pos);
  // The first and the last position of the wave's rows.
  const int pos_lo = wave_ok ? first + fdiv(wave_row, d.group_div) : 0;
  const int pos_hi = wave_ok ? first + fdiv(min(wave_row + 31, all_rows - 1), d.group_div) : -1;
  const int below_lo = sinks_only(d, pos_lo), below_hi = sinks_only(d, pos_hi);

  f16x8 q_hi[DP / 16], q_lo[DP / 16];
  float q_back;  // 1 / the row's power of two
  {
    const float* q = d.q + (int64_t)(w.start + token) * d.q_t + (int64_t)(w.head * d.group + sub) * d.q_h;
    float x[DP / 16][8], top = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 16; j++) {
      const int at = 16 * j + 8 * h;
      const bool ok = row_ok && at < dim;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 y = ok ? *(const float4*)(q + at + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[j][e] = y.x * d.scale_log2e, x[j][e + 1] = y.y * d.scale_log2e;
        x[j][e + 2] = y.z * d.scale_log2e, x[j][e + 3] = y.w * d.scale_log2e;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[j][e]));
    }
    const int q_up = exponent_for(half_max(top));
    const float f = pow2(q_up);
    q_back = pow2(-q_up);
#pragma unroll
    for (int j = 0; j < DP / 16; j++)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        f16x2 hi, lo;
        split16(x[j][e] * f, x[j][e + 1] * f, d.minus1, hi, lo);
        q_hi[j][e] = hi[0], q_hi[j][e + 1] = hi[1];
        q_lo[j][e] = lo[0], q_lo[j][e + 1] = lo[1];
      }
  }

  const int v_base = value_at<TN>(n, h);
  const Span span = span_of<TN>(d, w.kv_len, first + fdiv(row0, d.group_div),
                                first + fdiv(row0 + rows - 1, d.group_div));
  const int u0 = (int)((int64_t)span.tiles * w.part / w.parts), u1 = (int)((int64_t)span.tiles * (w.part + 1) / w.parts);
  const int* table = d.s.table + (int64_t)w.seq * d.s.table_stride;
  const char* kc = d.c.k + (int64_t)w.head * d.c.k_head * size;
  const char* vc = d.c.v + (int64_t)w.head * d.c.v_head * size;

  // Staging: wave w has keys 8 w .. 8 w + 7 of the tile, i = w & 1 of their 16;
  // of the keys a thread has an eighth of a row, of the values DP / 32
  // dimensions of four rows (h = half of the wave).
  struct Place {
    int k_row, k_eighth, v_group, v_chunk, v_half, v_key;
    __device__ explicit Place(int t)
        : k_row(t >> 3), k_eighth(t & 7), v_group(t & 31), v_chunk((t >> 7) * 2 + (t >> 5 & 1)), v_half(t >> 6 & 1),
          v_key(t >> 5 << 2) {}
  };
  // The rows of a tile: thread i < TN finds key i's page two tiles before the
  // loads need it and leaves its rows' offsets in LDS, the first row's where
  // nobody sees the key or it has no page.
  int page_next = -1;
  auto find_page = [&](int u) __attribute__((always_inline)) {
    page_next = -1;
    if (tid >= TN || u >= u1) return;
    const int key = span.tile(u) * TN + tid;
    if (key < span.end && (key >= span.lo || key < d.sinks)) page_next = page_entry(table, d.s.max_pages, d.c, key);
  };
  auto find_rows = [&](int u) __attribute__((always_inline)) {
    if (tid >= 64) return;
    const int key = (u < u1 ? span.tile(u) * TN : 0) + tid;
    const bool here = page_ok(d.c, page_next);
    const uint64_t all = __ballot(here);
    if (tid == 0) info_sh[u & 3].seen = all, info_sh[u & 3].bad = 0;
    if (tid >= TN) return;
    const int64_t slot = key - fdiv(key, d.c.page_div) * d.c.page_size;
    rows_sh[u & 3][0][tid] = here ? (page_next * d.c.k_page + slot * d.c.k_slot) * size : 0;
    rows_sh[u & 3][1][tid] = here ? (page_next * d.c.v_page + slot * d.c.v_slot) * size : 0;
  };
  u32x4 k_in[KL];
  uint32_t v_in[4][VW];
  auto load = [&](int u) __attribute__((always_inline)) {
    const Place at(afresh(tid));
    const char* kr = kc + rows_sh[u & 3][0][at.k_row];
#pragma unroll
    for (int j = 0; j < KL; j++) k_in[j] = *(const u32x4*)(kr + min((8 * j + at.k_eighth) * PER, dim - PER) * size);
#pragma unroll
    for (int r = 0; r < 4; r++)
      load_words<VW>(vc + rows_sh[u & 3][1][at.v_key + r], at.v_group * DPV * size, dim * size, v_in[r]);
  };

  float m, l;
  f32x16 o[NB];
  int o_up;  // o is 2^o_up times the result
  bool poison, uneven = false;
  // Converts the tile in the registers into its buffer.
  auto stage = [&](int u, auto with_care) __attribute__((always_inline)) {
    constexpr bool careful = decltype(with_care)::value;
    const int parity = u & 1;
    // Rows of keys that nobody sees.
    const uint64_t seen = info_sh[u & 3].seen;
    const uint32_t seen_lo = __builtin_amdgcn_readfirstlane((uint32_t)seen);
    const uint32_t seen_hi = __builtin_amdgcn_readfirstlane((uint32_t)(seen >> 32));
    if ((seen_lo & (TN == 64 ? seen_hi : ~0u)) != ~0u) {
      const Place p(afresh(tid));
      const bool k_here = seen >> p.k_row & 1;
#pragma unroll
      for (int j = 0; j < KL; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) k_in[j][e] = k_here ? k_in[j][e] : 0;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const bool v_here = seen >> (p.v_key + r) & 1;
#pragma unroll
        for (int c = 0; c < VW; c++) v_in[r][c] = v_here ? v_in[r][c] : 0;
      }
    }
    if constexpr (careful) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        bool bad = false;
#pragma unroll
        for (int c = 0; c < VW; c++) bad |= clean<TYPE>(v_in[r][c]);
        if (bad) atomicOr((unsigned long long*)&info_sh[u & 3].bad, 1ull << (Place(tid).v_key + r));
      }
    }
    float k_f = 1.f, v_f[4] = {1.f, 1.f, 1.f, 1.f};
    if constexpr (SCALED) {
      float k_top = 0.f, v_top[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (careful) {
#pragma unroll
        for (int j = 0; j < KL; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint32_t x = k_in[j][e];
            clean<TYPE>(x);
            k_top = top_of<TYPE>(k_top, x, 0);
          }
      } else {
#pragma unroll
        for (int j = 0; j < KL; j++)
#pragma unroll
          for (int e = 0; e < 4; e += 2) k_top = top_of<TYPE>(k_top, k_in[j][e], k_in[j][e + 1]);
      }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int c = 0; c < VW; c += 2) v_top[r] = top_of<TYPE>(v_top[r], v_in[r][c], c + 1 < VW ? v_in[r][c + 1] : 0);
      const uint32_t own = eighth_max(k_top);  // the lane's key's
      if constexpr (careful) {
        const int k_up = exponent_for(__uint_as_float(own));
        const Place at(tid);
        if (at.k_eighth == 0) key_up_sh[u & 3][at.k_row] = (int8_t)k_up;
        k_f = pow2(k_up);
      } else {
        // (A key of zeros has no bits to lose; 1 less, it is the largest of all.)
        const uint32_t top = wave_max_of_eighths(own), least = wave_min_of_eighths(own - 1);
        const int k_up = __builtin_amdgcn_readfirstlane(exponent_for(__uint_as_float(top)));
        if (lane == 0) {
          info_sh[u & 3].k_up[wave] = (int8_t)k_up;
          if (top >> 23 > (least >> 23) + EVEN) uneven_sh = 1;
        }
        k_f = pow2(k_up);
      }
      // (Of the values' tops the upper halves do: exponents and seven bits.)
      const auto two = [](float a, float b) {
        return half_max16(
            __builtin_bit_cast(u16x2, __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u)));
      };
      const u16x2 tops[2] = {two(v_top[0], v_top[1]), two(v_top[2], v_top[3])};
      const auto value_up = [](uint32_t top) {
        return top ? exponent_for(__uint_as_float(top << 16)) : NO_VALUE;
      };
      const auto factor = [](int up) { return up == NO_VALUE ? 0.f : pow2(up); };
      if constexpr (careful) {
        const Place at(tid);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int v_up = value_up(tops[r / 2][r % 2]);
          if (at.v_group == 0) value_up_sh[u & 3][at.v_key + r] = (int8_t)v_up;
          v_f[r] = factor(v_up);
        }
      } else {
        const auto other = [](u16x2 x) {
          const uint32_t y = __builtin_bit_cast(uint32_t, x);
          return __builtin_amdgcn_permlane32_swap(y, y, false, false);
        };
        const auto a = other(__builtin_elementwise_max(tops[0], tops[1]));
        const auto b = other(__builtin_elementwise_min(tops[0] - (uint16_t)1, tops[1] - (uint16_t)1));
        const u16x2 most = __builtin_elementwise_max(__builtin_bit_cast(u16x2, (uint32_t)a[0]),
                                                     __builtin_bit_cast(u16x2, (uint32_t)a[1]));
        const u16x2 least = __builtin_elementwise_min(__builtin_bit_cast(u16x2, (uint32_t)b[0]),
                                                      __builtin_bit_cast(u16x2, (uint32_t)b[1]));
        const uint32_t top = __builtin_amdgcn_readfirstlane(max((uint32_t)most[0], (uint32_t)most[1]));
        const int v_up = value_up(top);
        if (lane == 0) {
          info_sh[u & 3].v_up[wave] = (int8_t)v_up;
          if (top >> 7 > (min((uint32_t)least[0], (uint32_t)least[1]) >> 7) + EVEN) uneven_sh = 1;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) v_f[r] = factor(v_up);
      }
    }
    const Place p(afresh(tid));
    char* kt = &buffer_sh[parity][p.k_row * KS];
#pragma unroll
    for (int j = 0; j < KL; j++) {
      const int at = (8 * j + p.k_eighth) * PER * 2;
      if constexpr (TYPE == RTENHIP_CACHE_F16) {
        *(u32x4*)(kt + at) = k_in[j];
      } else if constexpr (TYPE == RTENHIP_CACHE_BF16) {
        u32x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++)
          y[e] = __builtin_bit_cast(uint32_t, (f16x2){(_Float16)(cache_lo<TYPE>(k_in[j][e]) * k_f),
                                                      (_Float16)(cache_hi<TYPE>(k_in[j][e]) * k_f)});
        *(u32x4*)(kt + at) = y;
      } else {
        f16x2 h0, l0, h1, l1;
        split16(__uint_as_float(k_in[j][0]), __uint_as_float(k_in[j][1]), k_f, k_f, h0, l0);
        split16(__uint_as_float(k_in[j][2]), __uint_as_float(k_in[j][3]), k_f, k_f, h1, l1);
        *(f16x4*)(kt + at) = (f16x4){h0[0], h0[1], h1[0], h1[1]};
        *(f16x4*)(kt + T::K_BYTES + at) = (f16x4){l0[0], l0[1], l1[0], l1[1]};
      }
    }
    char* vt = &buffer_sh[parity][TERMS * T::K_BYTES + 8 * p.v_half];
#pragma unroll
    for (int e = 0; e < DPV; e++) {
      const int at = value_at<TN>(DPV * p.v_group + e, p.v_chunk);
      if constexpr (TYPE == RTENHIP_CACHE_F16) {
        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
        *(u32x2*)(vt + at) = (u32x2){__builtin_amdgcn_perm(v_in[1][e / 2], v_in[0][e / 2], sel),
                                     __builtin_amdgcn_perm(v_in[3][e / 2], v_in[2][e / 2], sel)};
      } else if constexpr (TYPE == RTENHIP_CACHE_BF16) {
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; r++)
          x[r] = (e & 1 ? cache_hi<TYPE>(v_in[r][e / 2]) : cache_lo<TYPE>(v_in[r][e / 2])) * v_f[r];
        *(f16x4*)(vt + at) = (f16x4){(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
      } else {
        f16x2 h0, l0, h1, l1;
        split16(__uint_as_float(v_in[0][e]), __uint_as_float(v_in[1][e]), v_f[0], v_f[1], h0, l0);
        split16(__uint_as_float(v_in[2][e]), __uint_as_float(v_in[3][e]), v_f[2], v_f[3], h1, l1);
        *(f16x4*)(vt + at) = (f16x4){h0[0], h0[1], h1[0], h1[1]};
        *(f16x4*)(vt + T::V_BYTES + at) = (f16x4){l0[0], l0[1], l1[0], l1[1]};
      }
    }
  };
  // Gives o a smaller power of two.
  auto rescale = [&](int up) __attribute__((always_inline)) {
    const int to = max(up, O_LEAST), by = to - o_up;
    if (by >= 0) return;
    o_up = to;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[b][e] = __builtin_amdgcn_ldexpf(o[b][e], by);
  };
  auto multiply = [&](int u, auto with_care) __attribute__((always_inline)) {
    constexpr bool careful = decltype(with_care)::value;
    const int base = span.tile(u) * TN, parity = u & 1;
    // Tiles past all of the wave's rows, or before all their windows.
    if (!wave_ok || base > pos_hi || (base + TN - 1 <= below_lo && base >= d.sinks)) return;
    // (Read first and used after the first product, which does not need it.)
    const u32x4* from = (const u32x4*)&info_sh[u & 3];
    u32x4 ups = from[0], keys = from[1];
    bool whole = false;
    auto look = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        ups[i] = __builtin_amdgcn_readfirstlane(ups[i]), keys[i] = __builtin_amdgcn_readfirstlane(keys[i]);
      whole = (keys[0] & (TN == 64 ? keys[1] : ~0u)) == ~0u && !careful && wave_row + 31 < all_rows &&
              base + TN - 1 <= pos_lo && (base > below_hi || base + TN <= d.sinks);
      if constexpr (SCALED && !careful) {
        int least = NO_VALUE;
#pragma unroll
        for (int i = 0; i < WAVES; i++) least = min(least, (int)(int8_t)(ups[2 + i / 4] >> 8 * (i % 4)));
        if (least < o_up) rescale(least - 1);  // larger values than any before: a binade more of room
        uneven |= least < o_up;
      }
    };
    const char* ks = buffer_sh[parity];
    const char* vs = ks + TERMS * T::K_BYTES;
#pragma unroll 1
    for (int tb = 0; tb < TN / 32; tb++) {
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; e++) s[e] = 0.f;
      const char* kr = ks + (32 * tb + n) * KS + 16 * h;
      pipelined<DP / 16, AHEAD, Operands>(
          [&](int j) {
            Operands x;
#pragma unroll
            for (int i = 0; i < TERMS; i++) x.term[i] = *(const f16x8*)(kr + i * T::K_BYTES + 32 * j);
            return x;
          },
          [&](int j, const Operands& x) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[0], q_hi[j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[0], q_lo[j], s, 0, 0, 0);
            if constexpr (TERMS == 2) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[1], q_hi[j], s, 0, 0, 0);
          });
      if (tb == 0) look();
      if (!whole) {
        // (Without short circuits: a branch for each score costs the registers
        // of several copies of s.)
        const int half = afresh(lane) >> 5, at = base + 32 * tb + 4 * half;
        const uint32_t here = (tb ? keys[1] : keys[0]) >> 4 * half;
        uint32_t seen = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int k = (e & 3) + 8 * (e >> 2);  // at + k: the key of s[e]
          const bool ok = (here >> k & 1) & (at + k <= pos) & ((at + k > below) | (at + k < d.sinks));
          s[e] = ok ? s[e] : NEG_INF;
          seen |= (uint32_t)ok << k;
        }
        if (careful) poison |= (seen & (tb ? keys[3] : keys[2]) >> 4 * half) != 0;
      }
      // The factors of every 8 keys: of their scores, and of p.
      float back[4];
      int fall[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        back[i] = q_back;
        fall[i] = 0;
        if constexpr (SCALED) {
          // (Neither 0 nor infinity: a hidden score is -infinity, others may be 0.)
          const auto out_of = [&](int up) {
            return __builtin_amdgcn_fmed3f(q_back * pow2(-up), 1.17549435e-38f, 3.402823466e38f);
          };
          if constexpr (careful) {
            const uint32_t four = *(const uint32_t*)&key_up_sh[u & 3][32 * tb + 8 * i + 4 * h];
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * i + e] *= out_of((int8_t)(four >> 8 * e));
          } else {
            back[i] = out_of((int8_t)((tb ? ups[1] : ups[0]) >> 8 * i));
          }
          if constexpr (!careful) {
            const int up = (int8_t)((tb ? ups[3] : ups[2]) >> 8 * i);
            fall[i] = up == NO_VALUE ? 0 : max(o_up - up, -FALL);
            uneven |= up != NO_VALUE && o_up - up < -FALL;
          }
        }
      }
      if constexpr (careful) {  // the scores themselves
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (!SCALED) {
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * i + e] *= q_back;
          }
          back[i] = 1.f;
        }
      }
      float top = NEG_INF;
#pragma unroll
      for (int i = 0; i < 4; i++)
        top = fmaxf(top, fmaxf(fmaxf(s[4 * i], s[4 * i + 1]), fmaxf(s[4 * i + 2], s[4 * i + 3])) * back[i]);
      top = half_max(top);
      if (__any(careful ? top - m > 6.f : top > m + 6.f)) {
        const float m_new = fmaxf(m, top);
        // Neither 8 - m nor m + 6 is exact any more: with care the difference to
        // m is taken first.
        uneven |= fabsf(m_new) > 4194304.f && m_new != NEG_INF;
        const float fade = __builtin_amdgcn_exp2f(m - (m_new == NEG_INF ? 0.f : m_new));
        m = m_new;
        l *= fade;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int e = 0; e < 16; e++) o[b][e] *= fade;
      }
      // p 2^8: at most 2^14.
      const float m_of = m == NEG_INF ? 0.f : m, ref = 8.f - m_of;
      f16x8 p_hi[2], p_lo[2];
      if constexpr (SCALED && careful) {
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = __builtin_amdgcn_exp2f((s[e] - m_of) + 8.f), l += s[e];
        // The loudest values left and those within 2^FALL of them, until there
        // are none.
        const int own_up = value_up_sh[u & 3][32 * tb + n];
        uint32_t left = (uint32_t)__ballot(own_up != NO_VALUE);
        while (left) {
          const int up = __builtin_amdgcn_readfirstlane((int)wave_min(left >> n & 1 ? own_up + 128 : 255)) - 128;
          const uint32_t now = (uint32_t)__ballot((left >> n & 1) && own_up <= up + FALL);
          left &= ~now;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t four = *(const uint32_t*)&value_up_sh[u & 3][32 * tb + 8 * i + 4 * h];
            const uint32_t here = now >> (8 * i + 4 * h);
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
              p[e] = here >> e & 1 ? __builtin_amdgcn_ldexpf(s[4 * i + e], up - (int)(int8_t)(four >> 8 * e)) : 0.f;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              f16x2 hi, lo;
              split16(p[e], p[e + 1], d.minus1, hi, lo);
              const int at = 4 * (i & 1) + e;
              p_hi[i / 2][at] = hi[0], p_hi[i / 2][at + 1] = hi[1];
              p_lo[i / 2][at] = lo[0], p_lo[i / 2][at + 1] = lo[1];
            }
          }
          rescale(up - 1);
#pragma unroll
          for (int b = 0; b < NB; b++) {
            f32x16 t;
#pragma unroll
            for (int e = 0; e < 16; e++) t[e] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const int at = (v_base ^ value_flip<TN>(32 * b, 2 * (2 * tb + c))) + 32 * b * TN * 2;
              const f16x8 x = *(const f16x8*)(vs + at);
              t = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_hi[c], t, 0, 0, 0);
              t = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p_lo[c], t, 0, 0, 0);
              if constexpr (TERMS == 2)
                t = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const f16x8*)(vs + T::V_BYTES + at), p_hi[c], t, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) o[b][e] += __builtin_amdgcn_ldexpf(t[e], o_up - up);
          }
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float at = ref + (float)fall[i];
        float sum = 0.f;
#pragma unroll
        for (int e = 4 * i; e < 4 * i + 4; e += 2) {
          const float a = __builtin_amdgcn_exp2f(careful ? (s[e] - m_of) + 8.f : __fmaf_rn(s[e], back[i], at));
          const float b = __builtin_amdgcn_exp2f(careful ? (s[e + 1] - m_of) + 8.f : __fmaf_rn(s[e + 1], back[i], at));
          sum += a + b;
          f16x2 hi, lo;
          split16(a, b, d.minus1, hi, lo);
          p_hi[e >> 3][e & 7] = hi[0], p_hi[e >> 3][(e & 7) + 1] = hi[1];
          p_lo[e >> 3][e & 7] = lo[0], p_lo[e >> 3][(e & 7) + 1] = lo[1];
        }
        l = SCALED ? __fmaf_rn(sum, pow2(-fall[i]), l) : l + sum;
      }
      pipelined<2 * NB, AHEAD, Operands>(
          [&](int i) {
            const int c = i / NB, b = i % NB;
            const int at = (v_base ^ value_flip<TN>(32 * b, 2 * (2 * tb + c))) + 32 * b * TN * 2;
            Operands x;
#pragma unroll
            for (int k = 0; k < TERMS; k++) x.term[k] = *(const f16x8*)(vs + k * T::V_BYTES + at);
            return x;
          },
          [&](int i, const Operands& x) {
            const int c = i / NB, b = i % NB;
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[0], p_hi[c], o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[0], p_lo[c], o[b], 0, 0, 0);
            if constexpr (TERMS == 2) o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.term[1], p_hi[c], o[b], 0, 0, 0);
          });
    }
  };
  // A tile's buffer, tops and flags go by the parity of its number.
  auto pass = [&](auto careful) __attribute__((always_inline)) {
    m = NEG_INF, l = 0.f;
    o_up = 113;  // as for values that are all zero or very small
    poison = false;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[b][e] = 0.f;
    auto advance = [&](int u) __attribute__((always_inline)) {
      if (u + 1 < u1) stage(u + 1, careful);
      if (wave == 0) {
        find_rows(u + 3);
        find_page(u + 4);
      }
      load(u + 2);
    };
    if (tid == 0) uneven_sh = 0;
    find_page(u0);
    find_rows(u0);
    find_page(u0 + 1);
    find_rows(u0 + 1);
    find_page(u0 + 2);
    __syncthreads();
    load(u0);
    find_rows(u0 + 2);
    find_page(u0 + 3);
    stage(u0, careful);
    load(u0 + 1);
    for (int u = u0; u < u1; u++) {
      // Tile u is in its buffer, u + 2's rows are there, and nobody reads u - 1
      // any more.
      __syncthreads();
      if (WAVES == 4 || wave < 4) advance(u);
      multiply(u, careful);
      if (WAVES == 8 && wave >= 4) advance(u);
    }
    __syncthreads();
  };
  pass(std::false_type{});
  bool again = uneven || !finite(l);
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int e = 0; e < 16; e++) again |= !finite(o[b][e]);
  // (Seldom: what does not fit the registers is kept elsewhere there, not here.)
  if (__builtin_expect(__syncthreads_or((again && wave_ok) || uneven_sh) != 0, 0)) pass(std::true_type{});
  l = half_sum(l);
  if (half_max(poison ? 1.f : 0.f) > 0.f) l = __builtin_nanf("");
  if (!row_ok) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float v_back = SCALED ? pow2(-o_up) : 1.f;
  const int r = afresh(wave * 32 + n), to_token = fdiv(row0 + r, d.group_div), to_sub = row0 + r - to_token * d.group;
  float* to = w.slot < 0 ? d.out + (int64_t)(w.start + to_token) * d.o_t + (int64_t)(w.head * d.group + to_sub) * d.o_h
                         : d.o_big + ((int64_t)w.slot * T::ROWS + r) * dim;
  // (Without p's 2^14: results times weights of up to 1 are summed in 32 bits.)
  if (w.slot >= 0 && h == 0) d.ml_big[(int64_t)w.slot * T::ROWS + r] = make_float2(m, l * 0x1p-14f);
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int at = 32 * b + 2 * e + 4 * h;
      if (at < dim)
        *(f32x4*)(to + at) = (f32x4){o[b][e] * inv * v_back, o[b][e + 1] * inv * v_back, o[b][e + 2] * inv * v_back,
                                     o[b][e + 3] * inv * v_back};
    }
}

// ---- merge ---------------------------------------------------------------------------

__device__ __forceinline__ void join(float& m, float& l, f32x4& o, float m2, float l2, const f32x4& o2) {
  const float top = fmaxf(m, m2), ref = top == NEG_INF ? 0.f : top;
  const float a = __builtin_amdgcn_exp2f(m - ref), b = __builtin_amdgcn_exp2f(m2 - ref);
  m = top;
  l = __fmaf_rn(l, a, l2 * b);
#pragma unroll
  for (int e = 0; e < 4; e++) o[e] = __fmaf_rn(o[e], a, o2[e] * b);
}

constexpr int PA_MERGE_GRID = 512;  // workgroups; four times as many where chunk tiles may be cut
constexpr int PA_MERGE_BIG = 32;    // waves for a stretch's share of a chunk tile
constexpr int PA_MERGE_LEAST = 4;   // 16-byte pieces of a share

// out = sum_i l_i 2^(m_i - max m) o_i / sum_i l_i 2^(m_i - max m) over the
// stretches of a tile.  The stretches, which are as many slots, divide the
// tile's numbers among themselves, so a tile of many stretches is joined by
// many waves; where a share is short, several lanes take the stretches of a
// piece between them.  Bound by the latency of two dependent loads: 5 us for
// 64 sequences, of which 4 are any launch's; 11 us for a step of prompts and
// answers, all shares at once (15 us on 512 workgroups, in rounds).
__global__ __launch_bounds__(PA_THREADS) void merge_kernel(PagedDesc d) {
  const int n_small = d.slots_small ? d.slots[0] : 0, n_big = d.slots_big ? d.slots[1] : 0;
  const int units = n_small + n_big * PA_MERGE_BIG;
  const int lane = threadIdx.x & 63;
  const int dim = d.c.dim, quads = dim / 4;
  for (int unit = blockIdx.x * (PA_THREADS / 64) + (threadIdx.x >> 6); unit < units;
       unit += gridDim.x * (PA_THREADS / 64)) {
    const bool big = unit >= n_small;
    const int at_big = unit - n_small;
    const Part p = big ? d.part_big[at_big / PA_MERGE_BIG] : d.part_small[unit];
    const float* os = big ? d.o_big : d.o_small;
    const float2* ml = big ? d.ml_big : d.ml_small;
    const int tile_rows = big ? d.rows_big : PA_SMALL;
    const int slot0 = p.slot - p.part * p.stride;
    const int n = p.rows * quads;
    const int shares = big ? p.parts * PA_MERGE_BIG : p.parts;
    const int share = big ? p.part * PA_MERGE_BIG + at_big % PA_MERGE_BIG : p.part;
    const int each = max(PA_MERGE_LEAST, (n + shares - 1) / shares);
    const int begin = min(n, share * each), end = min(n, begin + each);
    if (begin >= end) continue;
    // Lanes for a piece: as many as leave a lane for every piece of the share.
    int lanes = 64;
    while (lanes > 1 && lanes * (end - begin) > 64) lanes >>= 1;
    const int first = lane & (lanes - 1);
    for (int at0 = begin; at0 < end; at0 += 64 / lanes) {
      const int at = at0 + lane / lanes, in = min(at, end - 1);
      const int row = in / quads, c = (in - row * quads) * 4;
      float m = NEG_INF, l = 0.f;
      f32x4 o = {0, 0, 0, 0};
#pragma unroll 4
      for (int i = first; i < p.parts; i += lanes) {
        const int64_t at_row = (slot0 + (int64_t)i * p.stride) * tile_rows + row;
        const float2 x = ml[at_row];
        f32x4 y = *(const f32x4*)(os + at_row * dim + c);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = x.y == 0.f ? 0.f : y[e] * x.y;
        join(m, l, o, x.x, x.y, y);
      }
      for (int k = 1; k < lanes; k <<= 1) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = __shfl_xor(o[e], k);
        const float m2 = __shfl_xor(m, k), l2 = __shfl_xor(l, k);
        join(m, l, o, m2, l2, y);
      }
      if (first == 0 && at < end) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= inv;
        const int r = p.row0 + row, token = fdiv(r, d.group_div), sub = r - token * d.group;
        *(f32x4*)(d.out + (int64_t)(p.token0 + token) * d.o_t + (int64_t)(p.head * d.group + sub) * d.o_h + c) = o;
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------

// Stretches that the decode kernel aims for, of which the card's 256 CUs hold
// `resident` workgroups: as many where the tiles are few, so that all run at
// once and end together; twice as many where there are many tiles, of lengths
// that differ, so that they even out (64 ragged sequences: 173 against 186 us
// with one each).
// The chunk kernel, one workgroup to a CU, aims for one each: its stretches'
// results are large, and joining twice as many costs more than they even out
// (prompts and answers mixed: 145 against 177 us in all).
static int decode_target(int resident, int64_t tiles) { return tiles * 2 <= resident ? resident : 2 * resident; }
constexpr int PA_TARGET_BIG = 256;

template <int DP>
constexpr int decode_waves() {
  return DecodeTile<DP, RTENHIP_CACHE_F32>::WAVES;
}

// Grids and workspace, from sizes the host knows.  A tile has its share of the
// target rounded, or one stretch: at most target + tiles in all, and where it
// has two or more at most 4 / 3 of its share.
struct PagedPlan {
  int64_t grid_small, grid_big, slots_small, slots_big;
  size_t bytes;
  int64_t slots, part_small, part_big, ml_small, ml_big, o_small, o_big;  // offsets in bytes
};

static rtenhip_status paged_plan(const rtenhip_tensor* q, const rtenhip_kv_cache* cache, const rtenhip_sequences* seqs,
                                 PagedDesc& d, int& dtype, PagedPlan& p) {
  if (!q) return fail(RTENHIP_MISSING_INPUTS, "Missing input");
  rtenhip_status st = cache_view(cache, d.c, dtype);
  if (st) return st;
  if (q->ndim != 3) return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Expected [tokens, heads, head_dim] inputs");
  const int64_t tokens = q->shape[0], heads = q->shape[1];
  if (tokens < 0 || heads < 1 || heads > 65536) return fail(RTENHIP_INVALID_VALUE, "Invalid input size");
  if (heads % d.c.heads)
    return fail(RTENHIP_INCOMPATIBLE_INPUT_SHAPES, "Query heads must be a multiple of the cache's");
  const int64_t group = heads / d.c.heads;
  // (Row numbers and grids stay below 2^31.)
  if (tokens * heads > (int64_t(1) << 30)) return fail(RTENHIP_UNSUPPORTED_VALUE, "Too many query rows");
  st = check_rows(q, tokens, heads, d.c.dim, "q must be [tokens, heads, head_dim] with the cache's head_dim",
                  "Head rows must have unit stride and start on 16 bytes");
  if (!st) st = seq_view(seqs, tokens, d.s);
  if (st) return st;
  d.group = (int)group;
  d.group_div = make_fastdiv((uint32_t)group);
  const int64_t n = seqs->n_seqs, hk = d.c.heads, dim = d.c.dim;
  d.rows_big = dim <= 64 ? chunk_rows<64>() : dim <= 128 ? chunk_rows<128>() : chunk_rows<256>();
  const int64_t longest = seqs->q_starts ? tokens : std::min<int64_t>(tokens, 1);  // new tokens of a sequence
  const bool small = group <= PA_SMALL, big = longest * group > PA_SMALL;
  // One stretch a tile where no sequence has more than one tile of keys.
  const bool splits = (int64_t)seqs->max_pages * cache->page_size > PA_UNIT;
  p = PagedPlan{};
  if (tokens && n) {
    const int64_t small_tiles = std::min(n, tokens) * hk;
    const int64_t big_tiles = (tokens * group / d.rows_big + std::min(n, tokens)) * hk;
    d.target_small = decode_target(256 * (dim <= 64 ? decode_waves<64>() : dim <= 128 ? decode_waves<128>() : decode_waves<256>()),
                                   small_tiles);
    d.target_big = PA_TARGET_BIG;
    if (small) p.grid_small = small_tiles + (splits ? d.target_small : 0);
    if (big) p.grid_big = big_tiles + (splits ? d.target_big : 0);
    if (!launchable(p.grid_small, PA_THREADS) || !launchable(p.grid_big, 2 * d.rows_big))
      return fail(RTENHIP_UNSUPPORTED_VALUE, "Too many query rows");
    if (splits) {
      p.slots_small = small ? d.target_small * 3 / 2 : 0;
      p.slots_big = big ? d.target_big * 3 / 2 : 0;
    }
  }
  size_t at = 0;
  const auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)((bytes + 255) / 256 * 256);
    return (int64_t)here;
  };
  if (splits) {
    p.slots = take(2 * (int64_t)sizeof(int));
    p.part_small = take(p.slots_small * (int64_t)sizeof(Part));
    p.part_big = take(p.slots_big * (int64_t)sizeof(Part));
    p.ml_small = take(p.slots_small * PA_SMALL * (int64_t)sizeof(float2));
    p.ml_big = take(p.slots_big * d.rows_big * (int64_t)sizeof(float2));
    p.o_small = take(p.slots_small * PA_SMALL * dim * 4);
    p.o_big = take(p.slots_big * d.rows_big * dim * 4);
  }
  p.bytes = at;
  return RTENHIP_OK;
}

// Whether the 16 keys of a decoding wave lie in one page, and distances within
// a page, and from one page to the next, fit 31 and 32 bits.  (64 ragged
// sequences of f32 rows: 311 us with pages of 16, 341 us with pages of 24,
// which are not; f16 176 and 179, bf16 of 64: 104 and 109.)
static bool decode_aligned(const CacheView& c, int size) {
  const int64_t in_page = (int64_t(1) << 31) / size / c.page_size, page = (int64_t(1) << 32) / size;
  return c.page_size % 16 == 0 && c.k_slot < in_page && c.v_slot < in_page && c.k_page < page && c.v_page < page;
}

template <int DP, int TYPE>
static void launch_paged(const PagedDesc& d, hipStream_t s) {
  const dim3 grid((unsigned)d.grid_small);
  if (d.grid_small && decode_aligned(d.c, CacheType<TYPE>::size))
    hipLaunchKernelGGL((decode_kernel<DP, TYPE, true>), grid, dim3(PA_THREADS), 0, s, d);
  else if (d.grid_small)
    hipLaunchKernelGGL((decode_kernel<DP, TYPE, false>), grid, dim3(PA_THREADS), 0, s, d);
  if (d.grid_big)
    hipLaunchKernelGGL((chunk_kernel<DP, TYPE>), dim3((unsigned)d.grid_big), dim3(ChunkTile<DP, TYPE>::THREADS), 0, s, d);
}

template <int TYPE>
static void launch_paged(const PagedDesc& d, hipStream_t s) {
  if (d.c.dim <= 64) launch_paged<64, TYPE>(d, s);
  else if (d.c.dim <= 128) launch_paged<128, TYPE>(d, s);
  else launch_paged<256, TYPE>(d, s);
}

}  // namespace rtenhip

using namespace rtenhip;

extern "C" rtenhip_status rtenhip_paged_attention_workspace(const rtenhip_tensor* q, const rtenhip_kv_cache* cache,
                                                            const rtenhip_sequences* seqs, size_t* bytes) {
  if (!bytes) return fail(RTENHIP_MISSING_INPUTS, "Missing output");
  PagedDesc d{};
  PagedPlan p;
  int dtype;
  const rtenhip_status st = paged_plan(q, cache, seqs, d, dtype, p);
  if (!st) *bytes = p.bytes;
  return st;
}

extern "C" rtenhip_status rtenhip_paged_attention_f32(rtenhip_ctx* ctx, const rtenhip_tensor* q,
                                                      const rtenhip_kv_cache* cache, const rtenhip_sequences* seqs,
                                                      float scale, int32_t window, int32_t sinks, void* workspace,
                                                      size_t workspace_bytes, rtenhip_tensor* out) {
  PagedDesc d{};
  PagedPlan p;
  int dtype;
  rtenhip_status st = paged_plan(q, cache, seqs, d, dtype, p);
  if (!st)
    st = check_rows(out, q->shape[0], q->shape[1], q->shape[2], "out must have the shape of q",
                    "Head rows must have unit stride and start on 16 bytes");
  if (st) return st;
  if (window < 0 || sinks < 0) return fail(RTENHIP_INVALID_VALUE, "window and sinks must not be negative");
  if (!std::isfinite(scale)) return fail(RTENHIP_INVALID_VALUE, "scale must be finite");
  if (!rows_apart(out->shape, out->strides, 2, q->shape[2]))
    return fail(RTENHIP_INVALID_VALUE, "Output rows must not overlap");
  if (rows_clash(q, out)) return fail(RTENHIP_INVALID_VALUE, "Outputs may share memory with their own input only");
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(RTENHIP_INVALID_VALUE, "Workspace is too small");
  if ((uintptr_t)workspace % 16) return fail(RTENHIP_UNSUPPORTED_VALUE, "Workspace must be on 16 bytes");
  if (!ctx) return fail(RTENHIP_MISSING_INPUTS, "Missing context");
  if (!p.grid_small && !p.grid_big) return RTENHIP_OK;
  d.q = q->data, d.q_t = q->strides[0], d.q_h = q->strides[1];
  if (d.c.n_pages == 0) {  // nothing to see, but a row to load: any of q's
    d.c.k = d.c.v = (char*)q->data;
    d.c.k_head = d.c.v_head = d.c.k_slot = d.c.v_slot = 0;
  }
  d.out = out->data, d.o_t = out->strides[0], d.o_h = out->strides[1];
  d.window = window;
  d.sinks = window ? sinks : 0;
  d.scale_log2e = scale * 1.44269504088896340736f;
  d.minus1 = -1.f;
  d.grid_small = (int)p.grid_small, d.grid_big = (int)p.grid_big;
  d.slots_small = (int)p.slots_small, d.slots_big = (int)p.slots_big;
  char* ws = (char*)workspace;
  if (p.bytes) {
    d.slots = (int*)(ws + p.slots);
    d.part_small = (Part*)(ws + p.part_small);
    d.part_big = (Part*)(ws + p.part_big);
    d.ml_small = (float2*)(ws + p.ml_small);
    d.ml_big = (float2*)(ws + p.ml_big);
    d.o_small = (float*)(ws + p.o_small);
    d.o_big = (float*)(ws + p.o_big);
  }
  DeviceScope on(reinterpret_cast<Ctx*>(ctx)->device);
  if (on.status) return on.status;
  hipStream_t s = stream_of(ctx);
  if (dtype == RTENHIP_CACHE_F32) launch_paged<RTENHIP_CACHE_F32>(d, s);
  else if (dtype == RTENHIP_CACHE_F16) launch_paged<RTENHIP_CACHE_F16>(d, s);
  else launch_paged<RTENHIP_CACHE_BF16>(d, s);
  RTENHIP_LAUNCH_CHECK();
  if (p.slots_small || p.slots_big) {
    hipLaunchKernelGGL(merge_kernel, dim3(p.slots_big ? 4 * PA_MERGE_GRID : PA_MERGE_GRID), dim3(PA_THREADS), 0, s, d);
    RTENHIP_LAUNCH_CHECK();
  }
  return RTENHIP_OK;
}
