// One token of each row of logits by temperature, top-k, top-p and min-p from a given uniform number, for
// gfx950: a workgroup a row. (Few rows stay in the dies' L2s between its passes; 256 of 131072 are read twice.)
//
// What top-k and top-p keep is a prefix of the row in descending order, ties by index. Weights are exp in 64
// bits, added as integers of 2^-s: such sums are exact and the same in any order, which atomics need, and with
// s = min(51, 62 - ceil(log2 V)) a row's sum is off by no more than 2^-(s + 1) an element, 3e-12 of the largest
// weight in all for V = 131072 in the mean.
//   top-k, up to 512   the k-th of the threads' own maxima is no more than the k-th of the row: one pass lists what is
//                      at least that (some 700 elements for 512), the list is sorted, the cuts are places in it, and
//                      sorted by place it gives the token
//   otherwise          a pass makes a histogram of the distance to the largest logit in 2048 steps, counts and
//                      weights; the next lists the elements of the steps in which the cuts lie and adds up the
//                      weight above them by tiles of the row; the cuts are found in the list digit by digit, and the
//                      token in the tile where the sum of what is kept passes uniform times all of it
//   rows of which too many elements share a step: the cuts digit by digit of the 32-bit keys, over the row
// Exponentials bound the passes: some 30 instructions an element, 40 us a pass for a row of 131072 in one workgroup.
// 1 row of 131072 by a sorted list takes 25 us, 64 by top-p 78 in parts (121 in one piece), 256 uncut 66.
// Where there are fewer rows than compute units, the passes of the second kind are launches of their own with
// several workgroups a row, which leave to the next what theirs have found, in memory of the call's own.
#include "decode_ops.h"
#include "dec_internal.h"

namespace dec {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kList = 4096, kTiles = 1024, kTable = 1024;
constexpr int kSorted = 512;            // top-k up to this by sorting a list
typedef unsigned long long u64;
constexpr float kNaN = __builtin_nanf("");
constexpr double kLog2e = 1.4426950408889634;
constexpr uint32_t kLowest = 0x007FFFFFu;       // key of -infinity

// Order-preserving bits of a float that is not NaN; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// The integers of a row's weights: 2^-51 at the finest, and the sum of V of them below 2^63.
__device__ __forceinline__ int unit_shift(int V) { return min(51, 62 - (V > 1 ? 32 - __clz(V - 1) : 0)); }

// 2^((x - top) rate) in units of 2^-shift, with rate = log2(e) / t. y = 1024 (x - top) rate = k + r, |r| <= 1/2: from
// a table of 2^(i / 1024), and 2^(r / 1024) - 1 as a polynomial whose first term left out, (r ln 2 / 1024)^4 / 24,
// is below 1e-15. k comes from the low bits of y + 1.5 2^52, and the rounding to an integer from adding 2^52.
struct Weights {
  float top;
  double rate, offset;                  // 1024 log2(e) / t, and top times it
  int shift;
  const double* table;
  __device__ __forceinline__ Weights(float top, double t, int shift, const double* table)
      : top(top), rate(1024.0 * kLog2e / t), offset((double)top * (1024.0 * kLog2e / t)), shift(shift), table(table) {}
  // in units, not rounded to whole ones, for x below top; less than half of one for -infinity
  __device__ __forceinline__ double units(float x) const {
    const double y = fmax(fma((double)x, rate, -offset), -1024.0 * 1000.0);
    const double k = y + 6755399441055744.0;
    const int n = (int)(uint32_t)__double_as_longlong(k);
    const double r = y - (k - 6755399441055744.0);
    const double q = r * fma(fma(r, 5.169222938345892e-11, 2.290978498068816e-07), r, 0.0006769015435155716);
    const u64 bits = (u64)__double_as_longlong(table[n & (kTable - 1)]);
    const double v = __longlong_as_double((long long)(bits + ((u64)((uint32_t)(n & -kTable) << 10) << 32)));
    return fma(v, q, v);
  }
  static __device__ __forceinline__ u64 whole(double units) {
    return (u64)__double_as_longlong(units + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const u64 w = whole(units(x));
    return x == top ? 1ull << shift : w;
  }
  // the weight where it is at least min_p, `least` in units (0: any)
  __device__ __forceinline__ u64 from(float x, double least) const {
    const double u = units(x);
    const u64 w = u >= least ? whole(u) : 0;
    return x == top ? 1ull << shift : w;
  }
};

struct Shared {
  double table[kTable];
  u64 mass[kBins];
  uint32_t count[kBins];
  uint32_t key[kList];                  // the list: keys and places
  int at[kList];
  u64 tile[kTiles];
  u64 wave[kWaves], wave2[kWaves];
  uint32_t listed;
};

// ---- over lanes and the workgroup ---------------------------------------------------------------
// (as instructions: fmaxf comes with one more an operand that makes signalling NaN quiet; rows with NaN have no token)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max4(const float x[4]) { return max3(max3(x[0], x[1], x[2]), x[3], x[3]); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 x) {
  return (u64)moved<CTRL, ROWS>((uint32_t)x) | (u64)moved<CTRL, ROWS>((uint32_t)(x >> 32)) << 32;
}
// (row_shr:1, 2, 4, 8, then the rows' last lanes: row_bcast:15 and 31)
#define ROW_STEPS STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF)
#define LANE_STEPS ROW_STEPS STEP(0x142, 0xA) STEP(0x143, 0xC)
// The value of lane ^ J.
template <int J>
__device__ __forceinline__ uint32_t across(uint32_t x) {
  if constexpr (J == 1) return moved<0xB1, 0xF>(x);                        // quad_perm:[1,0,3,2]
  else if constexpr (J == 2) return moved<0x4E, 0xF>(x);                   // quad_perm:[2,3,0,1]
  else if constexpr (J == 4) return moved<0x141, 0xF>(moved<0x1B, 0xF>(x));  // each four reversed, then each eight
  else if constexpr (J == 8) return moved<0x128, 0xF>(x);                  // row_ror:8
  else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);   // even rows' values, odd rows'
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int J>
__device__ __forceinline__ u64 across(u64 x) {
  return (u64)across<J>((uint32_t)x) | (u64)across<J>((uint32_t)(x >> 32)) << 32;
}
// Inclusive sums over the wave's lanes.
__device__ __forceinline__ u64 lane_sums(u64 x) {
#define STEP(ctrl, rows) x += moved<ctrl, rows>(x);
  LANE_STEPS
#undef STEP
  return x;
}
// The largest of the wave's lanes, in the last of them.
__device__ __forceinline__ u64 lane_max(u64 x) {
#define STEP(ctrl, rows) x = max(x, moved<ctrl, rows>(x));
  LANE_STEPS
#undef STEP
  return x;
}

static_assert(kWaves == 16, "a row of lanes has a value of each wave");
__device__ __forceinline__ u64 from_lane(u64 x, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane) << 32;
}
__device__ __forceinline__ int this_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// The largest of all threads.
__device__ __forceinline__ void all_max(Shared& s, u64& x, u64& y) {
  x = lane_max(x), y = lane_max(y);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave[threadIdx.x >> 6] = x, s.wave2[threadIdx.x >> 6] = y;
  __syncthreads();
  x = s.wave[threadIdx.x & 15], y = s.wave2[threadIdx.x & 15];
#define STEP(ctrl, rows) x = max(x, moved<ctrl, rows>(x)), y = max(y, moved<ctrl, rows>(y));
  ROW_STEPS
#undef STEP
  x = from_lane(x, 15), y = from_lane(y, 15);
}
__device__ __forceinline__ u64 all_max(Shared& s, u64 x) {
  u64 none = 0;
  all_max(s, x, none);
  return x;
}

// Sum of the threads before this one, and of all.
__device__ __forceinline__ void sums(Shared& s, u64 x, u64& before, u64& all) {
  const u64 up_to = lane_sums(x);
  const int wave = this_wave();
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave[wave] = up_to;
  __syncthreads();
  u64 waves = s.wave[threadIdx.x & 15];
#define STEP(ctrl, rows) waves += moved<ctrl, rows>(waves);
  ROW_STEPS
#undef STEP
  all = from_lane(waves, 15);
  before = up_to - x + (wave ? from_lane(waves, wave - 1) : 0);
}

// The values that the one thread with `mine` has (0 where none has), for all.
__device__ __forceinline__ void from_one(Shared& s, bool mine, u64& x, u64& y) {
  const int wave = this_wave();
  const bool here = __any(mine);
  __syncthreads();
  if (mine || (!here && (threadIdx.x & 63) == 0)) s.wave[wave] = mine ? x : 0, s.wave2[wave] = mine ? y : 0;
  __syncthreads();
  x = s.wave[threadIdx.x & 15], y = s.wave2[threadIdx.x & 15];
#define STEP(ctrl, rows) x |= moved<ctrl, rows>(x), y |= moved<ctrl, rows>(y);
  ROW_STEPS
#undef STEP
  x = from_lane(x, 15), y = from_lane(y, 15);
}
__device__ __forceinline__ u64 from_one(Shared& s, bool mine, u64 x) {
  u64 none = 0;
  from_one(s, mine, x, none);
  return x;
}

// Values in descending order, one a thread: a sorting network over the first `size` threads (a power of two, 64 at
// least; the others' values stay among themselves).
template <int J>
__device__ __forceinline__ u64 sorted_step(u64 x, int k) {
  const u64 y = across<J>(x);
  const bool larger = ((threadIdx.x & k) == 0) == ((threadIdx.x & J) == 0);
  return (x > y) == larger ? x : y;
}
__device__ __forceinline__ u64 sorted(Shared& s, u64 x, int size) {
  const int tid = threadIdx.x;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j >= 64; j >>= 1) {
      __syncthreads();
      s.mass[tid] = x;
      __syncthreads();
      const u64 y = s.mass[tid ^ j];
      const bool larger = ((tid & k) == 0) == ((tid & j) == 0);
      x = (x > y) == larger ? x : y;
    }
    if (k > 32) x = sorted_step<32>(x, k);
    if (k > 16) x = sorted_step<16>(x, k);
    if (k > 8) x = sorted_step<8>(x, k);
    if (k > 4) x = sorted_step<4>(x, k);
    if (k > 2) x = sorted_step<2>(x, k);
    x = sorted_step<1>(x, k);
  }
  __syncthreads();
  return x;
}
__device__ __forceinline__ int power_from(int n) {
  int size = 64;
  while (size < n) size <<= 1;
  return size;
}

// ---- the row ------------------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ float logit(const void* row, int i) {
  return BF16 ? bf16_f32(((const uint16_t*)row)[i]) : ((const float*)row)[i];
}

// A row in tiles of consecutive elements, a wave each in turn, in groups of 16 bytes a thread four times, loaded
// while the group before is worked on. Counted from the address of 16 bytes that the row begins in, `lead` elements
// before it; what is not of the row reads as -infinity. (Code stays small: with 32 elements of a thread unrolled, the
// passes waited for instructions, up to 1500 cycles an element of a wave.)
template <bool BF16>
struct Row {
  static constexpr int kRun = BF16 ? 8 : 4, kGroup = 64 * kRun * 4;
  const void* p;
  int V, lead, tile;                    // elements of a tile: kTiles of them hold the row
  int t0, end;                          // the first tile and the end of the elements of a sweep: of all, or of a part
  __device__ __forceinline__ Row(const void* p, int V) : p(p), V(V), lead((int)((uintptr_t)p % 16) / (BF16 ? 2 : 4)) {
    tile = kGroup;
    while ((long)tile * kTiles < (long)V + lead) tile <<= 1;
    t0 = 0, end = V;
  }
  // From here on, sweeps over one of `parts` parts.
  __device__ __forceinline__ void take_part(int part, int parts) {
    const int tiles = ((V + lead - 1) / tile + parts) / parts;
    t0 = part * tiles, end = (int)min((long)(part + 1) * tiles * tile - lead, (long)V);
  }
  __device__ __forceinline__ void load(uint4 (&u)[4], int from) const {
    const int at = from + (int)(threadIdx.x & 63) * kRun;
    const bool inside = from >= 0 && from + kGroup <= V;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int i = at + a * 64 * kRun;
      if (inside || (i >= 0 && i + kRun <= V)) {
        u[a] = BF16 ? *(const uint4*)((const uint16_t*)p + i) : *(const uint4*)((const float*)p + i);
      } else {
        constexpr uint32_t kNone = BF16 ? 0xFF80FF80u : 0xFF800000u;
        u[a] = {kNone, kNone, kNone, kNone};
        if (i < V && i + kRun > 0) {    // the row's ends: element by element, shifted in from above
#pragma unroll 1
          for (int j = i; j < i + kRun; ++j) {
            const bool in = j >= 0 && j < V;
            if constexpr (BF16) {
              const uint32_t x = in ? ((const uint16_t*)p)[j] : 0xFF80u;
              u[a] = {u[a].x >> 16 | u[a].y << 16, u[a].y >> 16 | u[a].z << 16, u[a].z >> 16 | u[a].w << 16,
                      u[a].w >> 16 | x << 16};
            } else {
              u[a] = {u[a].y, u[a].z, u[a].w, in ? ((const uint32_t*)p)[j] : kNone};
            }
          }
        }
      }
    }
  }
  // f(x, place) for four consecutive elements of this thread's in turn; done(tile) after each of its wave's tiles.
  template <bool LONG, typename F, typename G>
  __device__ __forceinline__ void sweep(const F& f, const G& done) const {
    int t = t0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), from = t * tile - lead;
    if (from >= end) return;
    uint4 u[4], next[4] = {};
    load(u, from);
#pragma unroll 1
    for (;;) {
      int then = from + kGroup;
      const bool last = then >= (t + 1) * tile - lead || then >= end;
      if (last) then = (t + kWaves) * tile - lead;
      if (then < end) load(next, then);
      const int at = from + (int)(threadIdx.x & 63) * kRun;
      // (one group of four elements in the code where f is long)
      const auto four = [&](const uint4 v, int i) {
        if constexpr (BF16) {
          uint32_t w0 = v.x, w1 = v.y;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            const float x[4] = {bf16_lo(w0), bf16_hi(w0), bf16_lo(w1), bf16_hi(w1)};
            f(x, i + 4 * half);
            w0 = v.z, w1 = v.w;
          }
        } else {
          const float x[4] = {bits_f32(v.x), bits_f32(v.y), bits_f32(v.z), bits_f32(v.w)};
          f(x, i);
        }
      };
      if constexpr (LONG) {
#pragma unroll 1
        for (int a = 0; a < 4; ++a) {
          four(u[0], at + a * 64 * kRun);
          u[0] = u[1], u[1] = u[2], u[2] = u[3];
        }
      } else {
#pragma unroll
        for (int a = 0; a < 4; ++a) four(u[a], at + a * 64 * kRun);
      }
      if (last) done(t), t += kWaves;
      if (then >= end) return;
      from = then;
#pragma unroll
      for (int a = 0; a < 4; ++a) u[a] = next[a];
    }
  }
  template <bool LONG, typename F>
  __device__ __forceinline__ void sweep(const F& f) const {
    sweep<LONG>(f, [](int) {});
  }
};

// Elements of a row with their weights, for find_cut.
template <typename R>
struct OfRow {
  const R& row;
  const Weights& w;
  template <typename F>
  __device__ __forceinline__ void each(const F& f) const {
    row.template sweep<true>([&](const float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f(key_of(x[j]), [&] { return w(x[j]); });
    });
  }
};
struct OfList {
  const Shared& s;
  int n;
  const Weights& w;
  template <typename F>
  __device__ __forceinline__ void each(const F& f) const {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t key = s.key[i];
      f(key, [&] { return w(of_key(key)); });
    }
  }
};

// The bin, of those that the threads have two each from the highest, in which the sum passes to `target` or more, and
// what lies above it. (~0: none.)
__device__ __forceinline__ uint32_t find_bin(Shared& s, const u64 m[2], u64 from, u64 target, u64& above) {
  u64 before, all;
  sums(s, m[0] + m[1], before, all);
  u64 x = from + before, hit = 0, at = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (x < target && x + m[j] >= target) hit = 2 * threadIdx.x + j + 1, at = x;
    x += m[j];
  }
  from_one(s, hit != 0, at, hit);
  above = at;
  return (uint32_t)hit - 1;
}

// The key at which the prefix of the order has `target` elements (BY_MASS: that much weight, over 0), digit by digit
// (11, 11 and 10 bits), and the elements and the weight above it. `count` and `mass` come with what lies above all
// elements of `from`.
template <bool BY_MASS, typename From>
__device__ __forceinline__ uint32_t find_cut(Shared& s, const From& from, u64 target, u64& count, u64& mass) {
  const int tid = threadIdx.x;
  uint32_t key = 0;
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
    const uint32_t fixed = level == 0 ? 0u : ~0u << (shift + bits);
    for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    from.each([&](uint32_t k, auto weight) {
      if ((k & fixed) != key) return;
      const uint32_t bin = (k >> shift) & ((1u << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], weight());
    });
    __syncthreads();
    u64 m[2], c[2], other;
#pragma unroll
    for (int j = 0; j < 2; ++j) m[j] = s.mass[kBins - 1 - 2 * tid - j], c[j] = s.count[kBins - 1 - 2 * tid - j];
    const uint32_t bin = find_bin(s, BY_MASS ? m : c, BY_MASS ? mass : count, target, other);
    // what lies above it by the other measure
    u64 before, all;
    const u64 mine0 = BY_MASS ? c[0] : m[0], mine1 = BY_MASS ? c[1] : m[1];
    sums(s, mine0 + mine1, before, all);
    const u64 up_to = from_one(s, bin >> 1 == (uint32_t)tid, before + (bin & 1 ? mine0 : 0));
    if (BY_MASS) mass = other, count += up_to;
    else count = other, mass += up_to;
    key |= (kBins - 1 - bin) << shift;
  }
  return key;
}

// ---- parameters ---------------------------------------------------------------------------------
struct Params {
  float t, p, mp;
  double least;                         // min-p in units
  int k;
  bool by_k, by_p;
  __device__ __forceinline__ Params(const SampleArgs& a, int row) {
    t = a.temperature ? a.temperature[row] : a.temperature_all;
    k = a.top_k ? a.top_k[row] : a.top_k_all;
    p = a.top_p ? a.top_p[row] : a.top_p_all;
    mp = a.min_p ? a.min_p[row] : a.min_p_all;
    least = mp > 0.0f ? ldexp((double)mp, unit_shift(a.V)) : 0.0;
    by_k = k >= 1 && k < a.V, by_p = p < 1.0f;
  }
  // the first of the largest, whatever the uniform number
  __device__ bool greedy() const { return !(t > 0.0f) || mp > 1.0f; }
  __device__ bool by_sorting() const { return by_k && k <= kSorted; }
  // how much weight top-p asks of `total`
  __device__ double asked(u64 total) const { return ceil((double)p * (double)total); }
};

// A cumulated sum exceeds uniform times all of it where it exceeds what whole number there is in that.
__device__ __forceinline__ u64 target_of(float uniform, u64 all) {
  const float u = fminf(fmaxf(uniform, 0.0f), 1.0f);
  return min((u64)((double)u * (double)all), all - 1);
}

// What is kept: keys above `key`, and those at it up to place `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool keeps(uint32_t k, int at) const { return k > key || (k == key && at <= last); }
};

// The place of the `ties`-th of the elements with this key, in order of places: 8 of its 24 bits at a time.
template <typename Each>
__device__ __forceinline__ int last_tie(Shared& s, u64 ties, const Each& each) {
  uint32_t at = 0;
#pragma unroll 1
  for (int shift = 16; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) s.count[i] = 0;
    __syncthreads();
    each([&](uint32_t place) {
      if (place >> (shift + 8) == at >> (shift + 8)) atomicAdd(&s.count[(place >> shift) & 255], 1u);
    });
    __syncthreads();
    const u64 c = threadIdx.x < 256 ? s.count[threadIdx.x] : 0;
    u64 before, all;
    sums(s, c, before, all);
    const bool hit = before < ties && before + c >= ties;
    u64 digit = threadIdx.x;
    from_one(s, hit, digit, before);
    at |= (uint32_t)digit << shift;
    ties -= before;
  }
  return (int)at;
}

// The token where tiles hold the kept weight of the row's tiles and weight(x, place) that of an element.
template <bool BF16, typename R, typename F>
__device__ __forceinline__ int locate(Shared& s, const R& row, float uniform, const F& weight) {
  u64 before, all;
  const u64 mine = s.tile[threadIdx.x];
  sums(s, mine, before, all);
  const u64 target = target_of(uniform, all);
  const bool hit = before <= target && before + mine > target;
  u64 where = threadIdx.x;
  from_one(s, hit, where, before);
  const int tile = (int)where;
  const u64 left = target - before;
  // runs of consecutive elements a thread
  const int run = row.tile / kThreads, to = (int)min((long)(tile + 1) * row.tile - row.lead, (long)row.V);
  const long i0 = (long)tile * row.tile - row.lead + (long)threadIdx.x * run;
  u64 sum = 0;
  for (int i = 0; i < run; ++i)
    if (i0 + i >= 0 && i0 + i < to) sum += weight(logit<BF16>(row.p, (int)i0 + i), (int)i0 + i);
  sums(s, sum, before, all);
  int at = -1;
  if (before <= left && before + sum > left) {
    u64 x = before;
    for (int i = 0; i < run && at < 0; ++i) {
      if (i0 + i >= 0 && i0 + i < to) x += weight(logit<BF16>(row.p, (int)i0 + i), (int)i0 + i);
      if (x > left) at = (int)i0 + i;
    }
  }
  return (int)from_one(s, at >= 0, (u64)(at + 1)) - 1;
}

// The weight of each tile into s.tile.
template <typename R, typename F>
__device__ __forceinline__ void weigh_tiles(Shared& s, const R& row, const F& weight) {
  s.tile[threadIdx.x] = 0;
  __syncthreads();
  u64 sum = 0;
  row.template sweep<true>([&](const float (&x)[4], int at) {
#pragma unroll
              for (int j = 0; j < 4; ++j) sum += weight(x[j], at + j);
            },
            [&](int t) {
              const u64 all = lane_sums(sum);
              if ((threadIdx.x & 63) == 63) s.tile[t] = all;
              sum = 0;
            });
  __syncthreads();
}

// top-k by sorting what is at least the k-th of the threads' maxima, or a little less; -2: too many.
template <typename R>
__device__ __forceinline__ int by_sorting(Shared& s, const R& row, const Params& par, const Weights& w, float uniform, float mine) {
  const int tid = threadIdx.x;
  // the lower end of the step, of 2048 from the largest of the threads' maxima to the least, that the k-th lies in
  const bool some = mine > -INFINITY;
  const float lowest = of_key(~(uint32_t)all_max(s, some ? ~key_of(mine) : 0u)), scale = 2047.0f / (w.top - lowest);
  const int step = mine == w.top ? 0 : (int)fminf((w.top - mine) * scale, 2047.0f);
  for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
  if (tid == 0) s.listed = 0;
  __syncthreads();
  if (some) atomicAdd(&s.count[step], 1u);
  __syncthreads();
  const u64 c[2] = {s.count[2 * tid], s.count[2 * tid + 1]};
  u64 above;
  const uint32_t bin = find_bin(s, c, 0, (u64)par.k, above);
  const uint32_t key = ~(uint32_t)all_max(s, some && (uint32_t)step <= bin ? ~key_of(mine) : 0u);
  const float least = of_key(bin == ~0u ? kLowest + 1 : key);
  row.template sweep<false>([&](const float (&x)[4], int at) {
    if (!(max4(x) >= least)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j)
      if (x[j] >= least) {
        const uint32_t i = atomicAdd(&s.listed, 1u);
        if (i < (uint32_t)kThreads) s.key[i] = key_of(x[j]), s.at[i] = at + j;
      }
  });
  __syncthreads();
  const int n = (int)s.listed;
  __syncthreads();                      // (by_steps clears it)
  if (n > kThreads) return -2;
  const int size = power_from(n);
  const u64 e = sorted(s, tid < n ? (u64)s.key[tid] << 32 | (uint32_t)~s.at[tid] : 0, size);
  const float x = of_key((uint32_t)(e >> 32));
  const bool there = tid < min(n, par.k);
  u64 weight = there ? w(x) : 0, before, all;
  sums(s, weight, before, all);
  const bool kept = there && (tid == 0 || (double)before < (par.by_p ? par.asked(all) : 1e300)) &&
                    w.from(x, par.least);
  // by place: ~place, descending
  const u64 f = sorted(s, kept ? (u64)(uint32_t)e << 32 | (uint32_t)(e >> 32) : 0, size);
  weight = f ? w(of_key((uint32_t)f)) : 0;
  sums(s, weight, before, all);
  const u64 target = target_of(uniform, all);
  const bool hit = before <= target && before + weight > target;
  return (int)from_one(s, hit, (u64)(~(uint32_t)(f >> 32)) + 1) - 1;
}

// Steps of the distance to the largest logit: 2046 over the finite logits, or over 48 t where that is less (what is
// further has 2^-69 of the weight, and is the last step).
struct Steps {
  float top, scale;
  bool some;
  __device__ __forceinline__ Steps(const Params& par, float top, float lowest) : top(top) {
    const float range = fminf(top - lowest, 48.0f * par.t);
    scale = 2046.0f / range, some = range > 0.0f && scale < 3e38f;
  }
  __device__ __forceinline__ int operator()(float x) const {
    return x == top ? 0 : (int)fminf((top - x) * scale, 2047.0f);
  }
};

// Counts and weights of the steps, where a cut asks for them.
template <typename R>
__device__ __forceinline__ void histogram(Shared& s, const R& row, const Params& par, const Weights& w, const Steps& step) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
  __syncthreads();
  row.template sweep<true>([&](const float (&x)[4], int) {
    u64 m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = w(x[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = step(x[j]);
      if (par.by_k && x[j] > -INFINITY) atomicAdd(&s.count[i], 1u);
      if (par.by_p && m[j]) atomicAdd(&s.mass[i], m[j]);
    }
  });
  __syncthreads();
}

// The steps to list, and what lies above them.
struct Span {
  bool by_k, by_p;
  uint32_t begin, end;
  u64 count, mass, all;                 // above `begin`; of the row
  Span() = default;
  // (m, c: the weights and counts of steps 2 tid and 2 tid + 1)
  __device__ __forceinline__ Span(Shared& s, const Params& par, const u64 m[2], const u64 c[2]) {
    const uint32_t tid = threadIdx.x;
    u64 before = 0, count_before = 0, elements = 0;
    all = 0;
    if (par.by_k) sums(s, c[0] + c[1], count_before, elements);
    if (par.by_p) sums(s, m[0] + m[1], before, all);
    by_k = par.by_k && elements > (u64)par.k, by_p = par.by_p;
    begin = end = kBins, count = mass = 0;            // no cut: none
    // That of the cut by top-k; that by top-p; with both all from the first in which the cut by top-p can be
    // (if nothing of top-k's step counts) to top-k's.
    if (by_k) {
      begin = end = find_bin(s, c, 0, (u64)par.k, count);
      mass = from_one(s, end >> 1 == tid, before + (end & 1 ? m[0] : 0));
    }
    if (by_p) {
      const double asked = par.asked(by_k ? mass : all);
      begin = find_bin(s, m, 0, (u64)fmax(asked, 1.0), mass);
      if (!by_k) end = begin;
      else count = from_one(s, begin >> 1 == tid, count_before + (begin & 1 ? c[0] : 0));
    }
  }
  __device__ __forceinline__ bool cuts() const { return by_k || by_p; }
  // (the last step is all that is further)
  __device__ __forceinline__ bool usable() const { return !cuts() || end < 2047; }
};

// The weight above the span by tiles to tile(t, sum), and the span's elements to list(key, place).
template <typename R, typename T, typename L>
__device__ __forceinline__ void survey(const R& row, const Params& par, const Weights& w, const Steps& step, const Span& span,
                                       const T& tile, const L& list) {
  u64 sum = 0;
  row.template sweep<true>(
      [&](const float (&x)[4], int at) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t i = (uint32_t)step(x[j]);
          const u64 m = w.from(x[j], par.least);
          if (i >= span.begin && i <= span.end) list(key_of(x[j]), at + j);     // (not -infinity, whose step is the last)
          sum += i < span.begin ? m : 0;
        }
      },
      [&](int t) {
        const u64 all = lane_sums(sum);
        if ((threadIdx.x & 63) == 63) tile(t, all);
        sum = 0;
      });
}

// The token, where s.tile holds the weight above the span by tiles, and s.key and s.at the span's n elements.
template <bool BF16, typename R>
__device__ __forceinline__ int by_list(Shared& s, const R& row, const Params& par, const Weights& w, float uniform, const Span& span,
                                       int n) {
  const int tid = threadIdx.x;
  const OfList list = {s, n, w};
  Cut cut = {0, 0x7FFFFFFF};
  if (span.cuts() && n <= kThreads) {
    // sorted, the cuts are places in it (3 us where the search digit by digit takes 13)
    const u64 e = sorted(s, tid < n ? (u64)s.key[tid] << 32 | (uint32_t)~s.at[tid] : 0, power_from(n));
    const float x = of_key((uint32_t)(e >> 32));
    const bool there = tid < n && (!span.by_k || span.count + tid < (u64)par.k);
    u64 before, all;
    sums(s, there ? w(x) : 0, before, all);
    const double asked = fmax(par.asked(span.by_k ? span.mass + all : span.all), 1.0);
    const bool kept = there && (!span.by_p || (double)(span.mass + before) < asked);
    const u64 last = ~all_max(s, kept ? ~e : 0);
    cut.key = (uint32_t)(last >> 32), cut.last = (int)~(uint32_t)last;
    if (kept) atomicAdd(&s.tile[((int)~(uint32_t)e + row.lead) / row.tile], w.from(x, par.least));
    __syncthreads();
  } else if (span.cuts()) {
    u64 ties = 0, total = span.all;
    if (span.by_k) {
      u64 count = span.count, mass = span.mass;
      cut.key = find_cut<false>(s, list, (u64)par.k, count, mass);
      ties = (u64)par.k - count;
      total = mass + ties * w(of_key(cut.key));
    }
    if (span.by_p) {
      u64 count = span.count, mass = span.mass;
      const u64 target = max((u64)fmax(par.asked(total), 1.0), mass + 1);
      if (target <= total) {
        cut.key = find_cut<true>(s, list, target, count, mass);
        const u64 each = max(w(of_key(cut.key)), 1ull);
        ties = (target - mass + each - 1) / each;
      }
    }
    cut.last = last_tie(s, ties, [&](auto f) {
      for (int i = tid; i < n; i += kThreads)
        if (s.key[i] == cut.key) f((uint32_t)s.at[i]);
    });
    for (int i = tid; i < n; i += kThreads) {
      const float x = of_key(s.key[i]);
      if (cut.keeps(s.key[i], s.at[i])) atomicAdd(&s.tile[(s.at[i] + row.lead) / row.tile], w.from(x, par.least));
    }
    __syncthreads();
  }
  return locate<BF16>(s, row, uniform, [&](float x, int at) -> u64 {
    return cut.keeps(key_of(x), at) ? w.from(x, par.least) : 0;
  });
}

// The weight of each tile to tile(t, sum), where nothing is cut.
template <typename R, typename T>
__device__ __forceinline__ void weigh(const R& row, const Params& par, const Weights& w, const T& tile) {
  u64 sum = 0;
  row.template sweep<true>(
      [&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += w.from(x[j], par.least);
      },
      [&](int t) {
        const u64 all = lane_sums(sum);
        if ((threadIdx.x & 63) == 63) tile(t, all);
        sum = 0;
      });
}

// top-k and top-p by steps; -2: too many in a step.
template <bool BF16, typename R>
__device__ __forceinline__ int by_steps(Shared& s, const R& row, const Params& par, const Weights& w, float uniform, float lowest) {
  const int tid = threadIdx.x;
  const Steps step(par, w.top, lowest);
  u64 m[2] = {}, c[2] = {};
  if (par.by_k || par.by_p) {
    if (!step.some) return -2;
    histogram(s, row, par, w, step);
#pragma unroll
    for (int j = 0; j < 2; ++j) m[j] = s.mass[2 * tid + j], c[j] = s.count[2 * tid + j];
  }
  const Span span(s, par, m, c);
  if (!span.usable()) return -2;
  s.tile[tid] = 0;
  if (tid == 0) s.listed = 0;
  __syncthreads();
  const auto tile = [&](int t, u64 sum) { s.tile[t] = sum; };
  if (!span.cuts())
    weigh(row, par, w, tile);
  else
    survey(row, par, w, step, span, tile, [&](uint32_t key, int at) {
      const uint32_t to = atomicAdd(&s.listed, 1u);
      if (to < (uint32_t)kList) s.key[to] = key, s.at[to] = at;
    });
  __syncthreads();
  const int n = (int)s.listed;
  return n > kList ? -2 : by_list<BF16>(s, row, par, w, uniform, span, n);
}

// The cuts digit by digit over the row.
template <bool BF16, typename R>
__device__ __forceinline__ int by_digits(Shared& s, const R& row, const Params& par, const Weights& w, float uniform) {
  Cut cut = {0, 0x7FFFFFFF};
  u64 ties = 0, count, mass, total = 0;
  bool some = false;
  const OfRow<R> from = {row, w};
  if (par.by_k) {
    count = mass = 0;
    cut.key = find_cut<false>(s, from, (u64)par.k, count, mass);
    ties = (u64)par.k - count, some = true;
    total = mass + ties * w(of_key(cut.key));
  }
  if (par.by_p) {
    if (!par.by_k) {
      u64 mine = 0, before;
      row.template sweep<true>([&](const float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += w(x[j]);
      });
      sums(s, mine, before, total);
    }
    const u64 target = (u64)fmax(par.asked(total), 1.0);
    if (target <= total) {
      count = mass = 0;
      cut.key = find_cut<true>(s, from, target, count, mass);
      const u64 each = max(w(of_key(cut.key)), 1ull);
      ties = (target - mass + each - 1) / each, some = true;
    }
  }
  if (some)
    cut.last = last_tie(s, ties, [&](auto f) {
      row.template sweep<true>([&](const float (&x)[4], int at) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
          if (key_of(x[j]) == cut.key) f((uint32_t)(at + j));
      });
    });
  const auto weight = [&](float x, int at) -> u64 {
    return cut.keeps(key_of(x), at) ? w.from(x, par.least) : 0;
  };
  weigh_tiles(s, row, weight);
  return locate<BF16>(s, row, uniform, weight);
}

// ---- a row in parts -----------------------------------------------------------------------------
// What the workgroups of a row's parts leave for the next launch.
struct PartOf {
  u64 top;                              // the key of the largest; ~0: there is a NaN
  u64 low;                              // ~ that of the lowest finite
  double sum;                           // of exp(x - top)
  uint32_t listed, pad;
  Span span;                            // of the row: the first part's
  u64 mass[kBins];
  uint32_t count[kBins];
  uint32_t key[kList];
  int at[kList];
};
__device__ __forceinline__ PartOf& part_of(const SampleArgs& a, int row, int part) {
  return ((PartOf*)((char*)a.workspace + (size_t)a.rows * kTiles * 8))[(size_t)row * a.parts + part];
}
__device__ __forceinline__ u64* tiles_of(const SampleArgs& a, int row) { return (u64*)a.workspace + (size_t)row * kTiles; }

template <bool BF16>
__device__ __forceinline__ Row<BF16> row_of(const SampleArgs& a, int at) {
  return Row<BF16>((const char*)a.logits + (size_t)at * a.row_stride * (BF16 ? 2 : 4), a.V);
}
__device__ __forceinline__ void fill_table(Shared& s, int V) {
  s.table[threadIdx.x] = exp2((double)threadIdx.x / kTable + unit_shift(V));   // (in units)
}
// A row's weights, over the table that this thread has filled its entry of. What the rounding of `offset` leaves out is
// the same for all of the row's exponents, and goes into the table where it is more than 2^-36, 2^-46 of a weight: from
// |top| / t of some 88. (From 1 on nothing else has weight: logits next to each other are 2^29 times as far apart.)
__device__ __forceinline__ Weights row_weights(Shared& s, float top, const Params& par, int V) {
  const Weights w(top, (double)par.t, unit_shift(V), s.table);
  const double rest = fma((double)top, w.rate, -w.offset);
  if (fabs(rest) > 0x1p-36 && fabs(rest) < 1.0) {
    s.table[threadIdx.x] *= exp2(-rest / kTable);
    __syncthreads();
  }
  return w;
}

// The largest, the lowest that is finite, each thread's largest and the first four elements that it is among.
struct Ends {
  float mine, low;
  int mine_at;
  u64 top_key, low_key;                 // of all threads; as in PartOf
  template <typename R>
  __device__ __forceinline__ Ends(Shared& s, const R& row, const Params& par) : mine(-INFINITY), low(INFINITY), mine_at(row.V) {
    bool bad = par.t != par.t;
    row.template sweep<false>([&](const float (&x)[4], int i) {
      bad |= __builtin_isunordered(x[0], x[1]) | __builtin_isunordered(x[2], x[3]);
      // (infinity times 0 is NaN, which a minimum passes by)
      low = min3(min3(low, fmaf(x[0], 0.0f, x[0]), fmaf(x[1], 0.0f, x[1])), fmaf(x[2], 0.0f, x[2]), fmaf(x[3], 0.0f, x[3]));
      const float m = max4(x);
      if (m > mine) mine = m, mine_at = i;
    });
    top_key = bad ? ~0u : key_of(mine), low_key = (uint32_t)~key_of(low);
    all_max(s, top_key, low_key);
  }
};
// Those of the parts, a lane each.
__device__ __forceinline__ void ends_of(const SampleArgs& a, int at, u64& top, u64& low) {
  top = low = 0;
  const int p = (int)(threadIdx.x & 15);
  top = low = 0;
  if (p < a.parts) top = part_of(a, at, p).top, low = part_of(a, at, p).low;
#define STEP(ctrl, rows) top = max(top, moved<ctrl, rows>(top)), low = max(low, moved<ctrl, rows>(low));
  ROW_STEPS
#undef STEP
  top = from_lane(top, 15), low = from_lane(low, 15);
}
// (~0 is the key of a NaN)
__device__ __forceinline__ bool has_token(u64 top) { return of_key((uint32_t)top) > -INFINITY; }

// The sum of exp(x - top): exponentials in fp32, a tile's sum of a thread in fp32. For thread 0.
template <typename R>
__device__ __forceinline__ double exp_sum(Shared& s, const R& row, float top) {
  const int tid = threadIdx.x;
  double sum = 0.0;
  float part = 0.0f;
  row.template sweep<true>(
      [&](const float (&x)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) part += x[j] == top ? 1.0f : __builtin_amdgcn_exp2f((x[j] - top) * 1.44269504f);
      },
      [&](int) { sum += (double)part, part = 0.0f; });
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  __syncthreads();
  if ((tid & 63) == 0) s.wave2[tid >> 6] = (u64)__double_as_longlong(sum);
  __syncthreads();
  sum = 0.0;
  if (tid == 0)
    for (int i = 0; i < kWaves; ++i) sum += __longlong_as_double((long long)s.wave2[i]);
  return sum;
}

// The counts and weights of steps 2 tid and 2 tid + 1 in all parts.
__device__ __forceinline__ void steps_of(const SampleArgs& a, int at, u64 m[2], u64 c[2]) {
#pragma unroll 4
  for (int p = 0; p < a.parts; ++p) {
    const PartOf& part = part_of(a, at, p);
#pragma unroll
    for (int j = 0; j < 2; ++j) m[j] += part.mass[2 * threadIdx.x + j], c[j] += part.count[2 * threadIdx.x + j];
  }
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_ends(SampleArgs a) {
  __shared__ Shared s;
  const int at = (int)blockIdx.x / a.parts, p = (int)blockIdx.x % a.parts;
  const Params par(a, at);
  if (par.greedy()) return;
  Row<BF16> row = row_of<BF16>(a, at);
  row.take_part(p, a.parts);
  const Ends ends(s, row, par);
  PartOf& part = part_of(a, at, p);
  if (threadIdx.x == 0) part.top = ends.top_key, part.low = ends.low_key;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_steps(SampleArgs a) {
  __shared__ Shared s;
  const int at = (int)blockIdx.x / a.parts, p = (int)blockIdx.x % a.parts, tid = threadIdx.x;
  const Params par(a, at);
  if (par.greedy()) return;
  u64 top_key, low_key;
  ends_of(a, at, top_key, low_key);
  if (!has_token(top_key)) return;
  const float top = of_key((uint32_t)top_key);
  Row<BF16> row = row_of<BF16>(a, at);
  row.take_part(p, a.parts);
  PartOf& part = part_of(a, at, p);
  const Steps step(par, top, of_key(~(uint32_t)low_key));
  if (step.some && (par.by_k || par.by_p)) {
    fill_table(s, a.V);
    const Weights w = row_weights(s, top, par, a.V);
    histogram(s, row, par, w, step);    // (its first barrier is the table's)
    for (int i = tid; i < kBins; i += kThreads) part.mass[i] = s.mass[i], part.count[i] = s.count[i];
  }
  if (a.logprobs) {
    const double sum = exp_sum(s, row, top);
    if (tid == 0) part.sum = sum;
  }
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_lists(SampleArgs a) {
  __shared__ Shared s;
  const int at = (int)blockIdx.x / a.parts, p = (int)blockIdx.x % a.parts, tid = threadIdx.x;
  const Params par(a, at);
  if (par.greedy()) return;
  u64 top_key, low_key;
  ends_of(a, at, top_key, low_key);
  if (!has_token(top_key)) return;
  const float top = of_key((uint32_t)top_key);
  const Steps step(par, top, of_key(~(uint32_t)low_key));
  u64 m[2] = {}, c[2] = {};
  if (par.by_k || par.by_p) {
    if (!step.some) return;
    steps_of(a, at, m, c);
  }
  fill_table(s, a.V);
  if (tid == 0) s.listed = 0;
  const Span span(s, par, m, c);
  if (p == 0 && tid == 0) part_of(a, at, 0).span = span;
  if (!span.usable()) return;
  __syncthreads();                      // (the table, and the list's length)
  const Weights w = row_weights(s, top, par, a.V);
  Row<BF16> row = row_of<BF16>(a, at);
  row.take_part(p, a.parts);
  PartOf& part = part_of(a, at, p);
  u64* const tiles = tiles_of(a, at);
  const auto tile = [&](int t, u64 sum) { tiles[t] = sum; };
  if (!span.cuts())
    weigh(row, par, w, tile);
  else
    survey(row, par, w, step, span, tile, [&](uint32_t key, int place) {
      const uint32_t to = atomicAdd(&s.listed, 1u);
      if (to < (uint32_t)kList) part.key[to] = key, part.at[to] = place;
    });
  __syncthreads();
  if (tid == 0) part.listed = s.listed;
}

// by_steps with what the parts' workgroups have left.
template <bool BF16, typename R>
__device__ __forceinline__ int by_parts(Shared& s, const SampleArgs& a, int at, const R& row, const Params& par, const Weights& w,
                                        float uniform, float lowest) {
  const int tid = threadIdx.x;
  if ((par.by_k || par.by_p) && !Steps(par, w.top, lowest).some) return -2;
  // (asked for together: what another die wrote is far)
  const Span span = part_of(a, at, 0).span;
  const int lane = tid & 63, wave = this_wave();
  const uint32_t listed = lane < a.parts ? part_of(a, at, lane).listed : 0;
  const u64 tile = (long)tid * row.tile < (long)row.V + row.lead ? tiles_of(a, at)[tid] : 0;
  if (!span.usable()) return -2;
  s.tile[tid] = tile;
  int n = 0;
  if (span.cuts()) {
    // a wave takes a part's list
    const u64 up_to = lane_sums((u64)listed);
    if (from_lane(up_to, 15) > (u64)kList) return -2;
    n = (int)from_lane(up_to, 15);
    if (wave < a.parts) {
      const PartOf& part = part_of(a, at, wave);
      const int to = (int)from_lane(up_to, wave), more = (int)from_lane((u64)listed, wave);
      for (int i = lane; i < more; i += 64) s.key[to - more + i] = part.key[i], s.at[to - more + i] = part.at[i];
    }
  }
  __syncthreads();
  return by_list<BF16>(s, row, par, w, uniform, span, n);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a) {
  __shared__ Shared s;
  const int at = blockIdx.x, tid = threadIdx.x;
  const Row<BF16> row = row_of<BF16>(a, at);
  const Params par(a, at);
  const bool in_parts = a.parts > 1 && !par.greedy();      // (rows that sort are one part)
  fill_table(s, a.V);
  float mine = 0.0f;
  int mine_at = row.V;
  u64 top_key, low_key;
  if (in_parts) {
    ends_of(a, at, top_key, low_key);
    __syncthreads();                    // (the table)
  } else {
    const Ends ends(s, row, par);
    mine = ends.mine, mine_at = ends.mine_at, top_key = ends.top_key, low_key = ends.low_key;
  }
  const float top = of_key((uint32_t)top_key);
  if (!has_token(top_key)) {
    if (tid == 0) {
      a.tokens[at] = -1;
      if (a.logprobs) a.logprobs[at] = kNaN;
    }
    return;
  }
  int token = -1;
  if (!par.greedy()) {
    const Weights w = row_weights(s, top, par, a.V);
    const float u = a.uniform[at], lowest = of_key(~(uint32_t)low_key);
    if (par.by_sorting()) token = by_sorting(s, row, par, w, u, mine);
    if (token < 0) token = in_parts ? by_parts<BF16>(s, a, at, row, par, w, u, lowest) : by_steps<BF16>(s, row, par, w, u, lowest);
    if (token < 0) token = by_digits<BF16>(s, row, par, w, u);
  }
  if (token < 0) {
    int place = 0x7FFFFFFF;
    for (int j = 3; j >= 0; --j) {
      const int i = mine_at + j;
      if (i >= 0 && i < row.V && logit<BF16>(row.p, i) == top) place = i;
    }
    token = (int)~(uint32_t)all_max(s, (uint32_t)~place);
  }
  if (a.logprobs) {
    double sum = 0.0;
    if (in_parts)
#pragma unroll 4
      for (int p = 0; p < a.parts; ++p) sum += part_of(a, at, p).sum;
    else
      sum = exp_sum(s, row, top);
    if (tid == 0) {
      const float x = logit<BF16>(row.p, token);
      a.logprobs[at] = (float)((x == top ? 0.0 : (double)x - (double)top) - log(sum));
    }
  }
  if (tid == 0) a.tokens[at] = token;
}

}  // namespace

// Into how many parts the rows go: so that there is a workgroup for each compute unit, with 16 of the smallest tiles
// each at least, one a wave; 16 parts at most, a lane and a wave of the last launch each. One part where every row goes
// by a sorted list, whose passes over the row take less than three launches, and where the rows have their own top_k
// (top_k 1 here): they may all sort. Those that do not pay for it, 1 (64) rows of 131072 with a top_k of 1000 take
// 89 us (91) where the number for all rows takes 35 (51).
int sample_parts(int rows, int V, bool bf16, int top_k) {
  if (rows < 1 || (top_k >= 1 && top_k <= kSorted && top_k < V)) return 1;
  return max(min(min(kCUs / rows, 16), V / (16 * (bf16 ? Row<true>::kGroup : Row<false>::kGroup))), 1);
}
size_t sample_workspace(int rows, int parts) {
  return parts > 1 ? (size_t)rows * (kTiles * 8 + (size_t)parts * sizeof(PartOf)) : 0;
}

namespace {
template <bool BF16>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
  if (a.parts > 1) {
    const int grid = a.rows * a.parts;
    const bool filters = a.top_p || (a.top_k_all >= 1 && a.top_k_all < a.V) || a.top_p_all < 1.0f;   // (top_k is null)
    sample_ends<BF16><<<grid, kThreads, 0, stream>>>(a);
    if (filters || a.logprobs) sample_steps<BF16><<<grid, kThreads, 0, stream>>>(a);
    sample_lists<BF16><<<grid, kThreads, 0, stream>>>(a);
  }
  sample_rows<BF16><<<a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  return a.bf16 ? launch<true>(a, stream) : launch<false>(a, stream);
}

}  // namespace dec
