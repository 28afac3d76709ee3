// One token of each row of logits by temperature, top-k, top-p and min-p from a given uniform number, for
// gfx950.
//
// What top-k and top-p keep is a prefix of the row in descending order, ties by index: all elements above a
// cut key and the first few at it. Weights are exp in 64 bits, added as integers of 2^-s: such sums are exact
// and the same in any order, which the atomics of a histogram need, and with s = 62 - ceil(log2 V) a row's sum
// is off by no more than 2^-(s + 1) an element, 3e-12 of the largest weight in all for V = 131072 in the mean.
//
// A row is read by as many workgroups as fill the card, twice:
//   survey    the largest logit, and how many elements and how much weight (against the largest value of the
//             bin, as the row's is not known yet) there are in each of 2048 bins of the keys' upper bits
//   collect   finds the bins in which the cut lies, adds up what is above them, and lists their elements
//   choose    one workgroup a row: the cut from the listed elements, digit by digit, then the part of the row
//             in which the sum of the kept weights passes uniform times their sum, and the token in it
// Without filters the row is read once (weigh, against the part's own largest logit, and pick). Rows of few
// elements, and those of which too many share a bin, are done by one workgroup (whole_row).
#include "decode_ops.h"
#include "dec_internal.h"

namespace dec {
namespace {

constexpr int kThreads = 1024, kBins = 2048, kBinShift = 21, kTile = 4096, kMaxTiles = 4096;
constexpr int kWide = 256;              // threads of the workgroups that share a row
constexpr int kCountBits = 14;          // of a bin's word in a workgroup: elements, at most 8192
constexpr int kRelative = 36;           // and weight above them, in 2^-36 of the bin's largest possible
typedef unsigned long long u64;
constexpr float kNaN = __builtin_nanf("");

// Order-preserving bits of a float that is not NaN; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// 2^(y + scale) in 64 bits, y <= 0: 2^(k / 64) from a table, and a polynomial for the rest x of at most 2^-7 (the
// first term left out, (x ln 2)^5 / 120, is below 4e-14).
__device__ __forceinline__ double exp2_64(double y, const double* table, int scale = 0) {
  const double k = __builtin_rint(fmax(y, -1100.0) * 64.0);
  const double x = fma(k, -0.015625, fmax(y, -1100.0));
  const int n = (int)k;
  double p = fma(x, 0.009618129107628477, 0.05550410866482158);
  p = fma(p, x, 0.24022650695910072);
  p = fma(p, x, 0.6931471805599453);
  p = fma(p, x, 1.0);
  return __builtin_ldexp(table[n & 63] * p, (n >> 6) + scale);
}
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
}
// x of 0 .. 2^52 - 1 rounded to an integer: the low bits of 2^52 + x.
__device__ __forceinline__ u64 to_units(double x) {
  return (u64)__double_as_longlong(x + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}

struct Weights {
  float top;
  double rate;                          // log2(e) / t
  int shift;                            // integers of 2^-shift
  const double* table;
  __device__ double real(float x) const {
    return x == top ? 1.0 : exp2_64(((double)x - (double)top) * rate, table);
  }
  __device__ u64 operator()(float x) const {
    if (x == top) return 1ull << shift;
    return x == -INFINITY ? 0 : to_units(exp2_64(((double)x - (double)top) * rate, table, shift));
  }
  // the weight where it is at least min_p (over 0)
  __device__ u64 at_least(float x, float min_p) const {
    return min_p > 0.0f && !(real(x) >= (double)min_p) ? 0 : (*this)(x);
  }
};
constexpr double kLog2e = 1.4426950408889634;
// The integers of a row's weights: 2^-51 at the finest, and the sum of V of them below 2^63.
__device__ __forceinline__ int unit_shift(int V) { return min(51, 62 - (V > 1 ? 32 - __clz(V - 1) : 0)); }

struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 wave_mass[16];
  uint32_t wave_count[16];
  u64 tile_mass[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  double table[64];
  uint32_t key, index;
  u64 above_count, above_mass;
  int flag, found;
};

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ uint32_t lane_sums(uint32_t x) {
#define STEP(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, false);
  STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF) STEP(0x142, 0xA) STEP(0x143, 0xC)
#undef STEP
  return x;
}
__device__ __forceinline__ u64 lane_sums(u64 x) {
#define STEP(ctrl, rows)                                                                                        \
  x += (u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, ctrl, rows, 0xF, false) |                \
       (u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), ctrl, rows, 0xF, false) << 32;
  STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF) STEP(0x142, 0xA) STEP(0x143, 0xC)
#undef STEP
  return x;
}

// Sums of the threads before this one, and of all.
template <int N>
__device__ void scan(u64* wave_mass, uint32_t* wave_count, u64 m, uint32_t c, u64& before_m, uint32_t& before_c,
                     u64& all_m) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 im = lane_sums(m);
  const uint32_t ic = lane_sums(c);
  __syncthreads();
  if (lane == 63) wave_mass[wave] = im, wave_count[wave] = ic;
  __syncthreads();
  before_m = im - m, before_c = ic - c, all_m = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    if (w < wave) before_m += wave_mass[w], before_c += wave_count[w];
    all_m += wave_mass[w];
  }
}
__device__ __forceinline__ void scan(Shared& s, u64 m, uint32_t c, u64& before_m, uint32_t& before_c, u64& all_m) {
  scan<kThreads>(s.wave_mass, s.wave_count, m, c, before_m, before_c, all_m);
}

template <bool BF16>
__device__ __forceinline__ float logit(const void* row, int i) {
  return BF16 ? bf16_f32(((const uint16_t*)row)[i]) : ((const float*)row)[i];
}

// A row's parameters.
struct Params {
  float t, p, mp;
  int k;
  bool by_k, by_p;
  __device__ Params(const SampleArgs& a, int row) {
    t = a.temperature ? a.temperature[row] : a.temperature_all;
    k = a.top_k ? a.top_k[row] : a.top_k_all;
    p = a.top_p ? a.top_p[row] : a.top_p_all;
    mp = a.min_p ? a.min_p[row] : a.min_p_all;
    by_k = k >= 1 && k < a.V, by_p = p < 1.0f;
  }
  // the first of the largest, whatever the uniform number
  __device__ bool greedy() const { return !(t > 0.0f) || mp > 1.0f; }
};
__device__ __forceinline__ const void* row_of(const SampleArgs& a, int row) {
  return (const char*)a.logits + (size_t)row * a.row_stride * (a.bf16 ? 2 : 4);
}
__device__ __forceinline__ u64 target_of(float uniform, u64 Z) {
  // (a cumulated sum exceeds u Z where it exceeds what whole number there is in u Z)
  const float u = fminf(fmaxf(uniform, 0.0f), 1.0f);
  return min((u64)((double)u * (double)Z), Z - 1);
}

// The cut at which the prefix of the order has `target` elements (BY_MASS: that much weight, > 0): its key,
// and what lies above the key. Element i < n has at.key(i) and at.weight(i); `key` comes with the bits of the
// digits before `level`, which all elements that can be at the cut share.
template <bool BY_MASS, typename Source>
__device__ void find_cut(Shared& s, int n, const Source& at, u64 target, uint32_t& key, u64& above_count,
                         u64& above_mass, int level = 0) {
  const int tid = threadIdx.x;
  for (; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
    const uint32_t fixed = level == 0 ? 0u : ~0u << (shift + bits);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = at.key(i);
      if ((k & fixed) != key) continue;
      const uint32_t bin = (k >> shift) & ((1u << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], at.weight(i));
    }
    __syncthreads();
    u64 m[2], before_m, all_m;
    uint32_t c[2], before_c;
    for (int j = 0; j < 2; ++j) m[j] = s.mass[kBins - 1 - 2 * tid - j], c[j] = s.count[kBins - 1 - 2 * tid - j];
    scan(s, m[0] + m[1], c[0] + c[1], before_m, before_c, all_m);
    u64 am = above_mass + before_m, ac = above_count + before_c;
    for (int j = 0; j < 2; ++j) {
      const u64 x = BY_MASS ? am : ac, more = BY_MASS ? m[j] : (u64)c[j];
      if (x < target && x + more >= target)
        s.key = key | (uint32_t)(kBins - 1 - 2 * tid - j) << shift, s.above_count = ac, s.above_mass = am;
      am += m[j], ac += c[j];
    }
    __syncthreads();
    key = s.key, above_count = s.above_count, above_mass = s.above_mass;
  }
}

template <bool BF16>
struct RowSource {
  const void* row;
  const Weights& w;
  __device__ uint32_t key(int i) const { return key_of(logit<BF16>(row, i)); }
  __device__ u64 weight(int i) const { return w(logit<BF16>(row, i)); }
};

// A row in one workgroup.
template <bool BF16>
__device__ void whole_row(const SampleArgs& a, int row_at, Shared& s) {
  const int tid = threadIdx.x, V = a.V;
  const void* row = row_of(a, row_at);
  const Params par(a, row_at);
  const float t = par.t, mp = par.mp;
  __syncthreads();
  fill_table(s.table);

  // the largest logit and where it is first
  uint32_t top = 0, at = 0xFFFFFFFFu;
  bool bad = t != t;
  for (int i = tid; i < V; i += kThreads) {
    const float x = logit<BF16>(row, i);
    bad |= x != x;
    const uint32_t key = x != x ? 0 : key_of(x);
    if (key > top) top = key, at = i;
  }
  if (tid == 0) s.key = 0, s.index = 0xFFFFFFFFu, s.flag = 0, s.found = -1;
  __syncthreads();
  atomicMax(&s.key, top);
  if (bad) s.flag = 1;
  __syncthreads();
  if (top == s.key) atomicMin(&s.index, at);
  __syncthreads();
  const Weights w = {of_key(s.key), kLog2e / (double)t, unit_shift(V), s.table};
  const int first = (int)s.index;
  const bool none = s.flag || w.top == -INFINITY;
  if (none) {
    if (tid == 0) {
      a.tokens[row_at] = -1;
      if (a.logprobs) a.logprobs[row_at] = kNaN;
    }
    return;
  }
  int token = first;
  if (!par.greedy()) {
    uint32_t cut = 0;                   // kept: keys above it, and the first `ties` at it
    u64 ties = 0, above_count = 0, above_mass = 0;
    const bool by_k = par.by_k, by_p = par.by_p;
    const RowSource<BF16> source = {row, w};
    u64 total = 0;
    if (by_k) {
      find_cut<false>(s, V, source, (u64)par.k, cut, above_count, above_mass);
      ties = (u64)par.k - above_count;
      total = above_mass + ties * w(of_key(cut));
    }
    if (by_p) {
      if (!by_k) {
        u64 mine = 0, before;
        uint32_t c;
        for (int i = tid; i < V; i += kThreads) mine += w(logit<BF16>(row, i));
        scan(s, mine, 0, before, c, total);
      }
      const double want = ceil((double)par.p * (double)total);
      if (want >= 1.0) {
        const u64 target = min((u64)want, total);
        above_count = above_mass = cut = 0;
        find_cut<true>(s, V, source, target, cut, above_count, above_mass);
        const u64 each = w(of_key(cut));
        ties = (target - above_mass + each - 1) / each;
      } else {
        cut = key_of(w.top), ties = 1;
      }
    }
    // kept weight and ties of each tile, in index order
    const int tile = max(kTile, (ceil_div(V, kMaxTiles) + kThreads - 1) / kThreads * kThreads);
    const auto weight = [&](float x, uint32_t& tie) -> u64 {
      const uint32_t key = key_of(x);
      tie = key == cut && (by_k || by_p);
      return key < cut ? 0 : w.at_least(x, mp);
    };
    for (int i = tid; i < kMaxTiles; i += kThreads) s.tile_mass[i] = 0, s.tile_ties[i] = 0;
    __syncthreads();
    for (int t0 = 0, n = 0; t0 < V; t0 += tile, ++n) {
      u64 m = 0;
      uint32_t c = 0;
      for (int i = t0 + tid; i < min(V, t0 + tile); i += kThreads) {
        uint32_t tie;
        const u64 x = weight(logit<BF16>(row, i), tie);
        c += tie;
        if (!tie) m += x;
      }
      for (int d = 32; d; d >>= 1) m += __shfl_xor(m, d), c += __shfl_xor(c, d);
      if ((tid & 63) == 0) atomicAdd(&s.tile_mass[n], m), atomicAdd(&s.tile_ties[n], c);
    }
    __syncthreads();
    const int tiles = ceil_div(V, tile);
    uint32_t unused;
    const u64 each = by_k || by_p ? weight(of_key(cut), unused) : 0;
    u64 Z = 0, left = ties;
    for (int n = 0; n < tiles; ++n) {
      const u64 here = min((u64)s.tile_ties[n], left);
      Z += s.tile_mass[n] + here * each, left -= here;
    }
    const u64 target = target_of(a.uniform[row_at], Z);
    u64 sum = 0;
    left = ties;
    int n = 0;
    for (; n < tiles; ++n) {
      const u64 here = min((u64)s.tile_ties[n], left), next = sum + s.tile_mass[n] + here * each;
      if (next > target) break;
      sum = next, left -= here;
    }
    // the token inside that tile, a round of kThreads elements at a time
    for (int t0 = n * tile; t0 < min(V, (n + 1) * tile) && s.found < 0; t0 += kThreads) {
      const int i = t0 + tid;
      uint32_t tie = 0, ties_before, c;
      u64 x = 0, before, all;
      if (i < min(V, (n + 1) * tile)) x = weight(logit<BF16>(row, i), tie);
      scan(s, 0, tie, before, ties_before, all);
      if (tie && ties_before >= left) x = 0;
      scan(s, x, tie, before, c, all);
      if (x && sum + before <= target && sum + before + x > target) s.found = i;
      if (tid == kThreads - 1) s.index = c + tie;
      __syncthreads();
      sum += all, left -= min((u64)s.index, left);
      __syncthreads();
    }
    __syncthreads();
    token = s.found;
  }
  if (a.logprobs) {
    const Weights one = {w.top, kLog2e, w.shift, s.table};
    u64 mine = 0, before, total;
    uint32_t c;
    for (int i = tid; i < V; i += kThreads) mine += one(logit<BF16>(row, i));
    scan(s, mine, 0, before, c, total);
    if (tid == 0) {
      const float x = logit<BF16>(row, token);
      a.logprobs[row_at] =
          (float)((x == w.top ? 0.0 : (double)x - (double)w.top) - log(ldexp((double)total, -w.shift)));
    }
  }
  if (tid == 0) a.tokens[row_at] = token;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a) {
  __shared__ Shared s;
  whole_row<BF16>(a, blockIdx.x, s);
}

// ---- a row shared by workgroups -----------------------------------------------------------------
// What a workgroup found in its part of a row.
struct Part {
  u64 kept;                             // weight above the listed bins (weigh: of all, against `top`)
  u64 near;                             // weight of the bin of `top`, against it
  double sum;                           // for log probabilities: of exp(x - top)
  uint32_t top;                         // key of the largest
  int at;                               // and its first place
  int bad, pad;                         // NaN among them
};
struct Entry {
  u64 weight;
  uint32_t key;
  int at;
};
// A row's part of the workspace, followed by its parts and its list.
struct RowSpace {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 below, above_count;               // weight of the bins below those listed, elements above them
  uint32_t listed, low, high;           // entries of the list; keys of its bins, low <= key < high
  uint32_t by_k;                        // there are top_k elements
};
struct Layout {
  int per, parts, most;                 // elements of a part, parts, entries of the list
  size_t list, row;                     // offsets in a row's space, and its size
};
__host__ __device__ inline Layout layout_of(int rows, int V, bool filters) {
  Layout l;
  l.per = (long)rows * ((V + 8191) / 8192) >= 2 * kCUs || V > 2048 * kMaxTiles ? 8192 : 2048;
  l.parts = (V + l.per - 1) / l.per;
  l.most = filters ? min(V, max(16384, V / 8)) : 0;
  l.list = (filters ? sizeof(RowSpace) : 0) + l.parts * sizeof(Part);
  l.row = l.list + (size_t)l.most * sizeof(Entry);
  return l;
}

struct Shape {
  Layout l;
  bool filters;
  __device__ char* row(const SampleArgs& a, int r) const { return (char*)a.workspace + r * l.row; }
  __device__ RowSpace& space(const SampleArgs& a, int r) const { return *(RowSpace*)row(a, r); }
  __device__ Part* parts(const SampleArgs& a, int r) const { return (Part*)(row(a, r) + (filters ? sizeof(RowSpace) : 0)); }
  __device__ Entry* list(const SampleArgs& a, int r) const { return (Entry*)(row(a, r) + l.list); }
};

__global__ __launch_bounds__(kWide) void clear_rows(SampleArgs a, Shape sh) {
  u64* p = (u64*)sh.row(a, blockIdx.x);
  for (unsigned i = threadIdx.x; i < sizeof(RowSpace) / 8; i += kWide) p[i] = 0;
}

// The elements that a thread has of its workgroup's part, N of them, -infinity past the end. VEC: 16 bytes
// at a time from aligned rows.
template <bool BF16, bool VEC, int N>
struct Mine {
  float x[N];
  int base, step;                       // places of the first, and from one run to the next
  static constexpr int kRun = VEC ? (BF16 ? 8 : 4) : 1;
  __device__ void load(const void* row, int from, int V) {
    base = from + (int)threadIdx.x * kRun;
    step = kWide * kRun;
#pragma unroll
    for (int i = 0; i < N; i += kRun) {
      const int at = place(i);
      if constexpr (VEC) {
        if (at + kRun <= V) {
          const uint4 u = BF16 ? *(const uint4*)((const uint16_t*)row + at) : *(const uint4*)((const float*)row + at);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (BF16) x[i + 2 * j] = bf16_lo(w[j]), x[i + 2 * j + 1] = bf16_hi(w[j]);
            else x[i + j] = __uint_as_float(w[j]);
          }
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < kRun; ++j) x[i + j] = at + j < V ? logit<BF16>(row, at + j) : -INFINITY;
    }
  }
  __device__ int place(int i) const { return base + i / kRun * step + i % kRun; }
};

struct WideShared {
  u64 bins[kBins];
  u64 wave_mass[4];
  uint32_t wave_count[4];
  double table[64], wave_sum[4];
  uint32_t top, at;
  int bad;
};

// The part's largest logit and first place, and whether it holds NaN; returns the key.
template <typename M, int N>
__device__ uint32_t largest(WideShared& s, const M& m, Part& part) {
  if (threadIdx.x == 0) s.top = 0, s.at = 0xFFFFFFFFu, s.bad = 0;
  uint32_t top = 0, at = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    bad |= m.x[i] != m.x[i];
    const uint32_t k = m.x[i] != m.x[i] ? 0 : key_of(m.x[i]);
    if (k > top) top = k, at = (uint32_t)m.place(i);
  }
  uint32_t most = top;
  for (int d = 32; d; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) atomicMax(&s.top, most);
  if (__any(bad) && (threadIdx.x & 63) == 0) s.bad = 1;
  __syncthreads();
  if (top == s.top) atomicMin(&s.at, at);
  __syncthreads();
  part.top = s.top, part.at = (int)s.at, part.bad = s.bad;
  return s.top;
}

// Sum over the workgroup in a fixed order.
__device__ __forceinline__ double sum_all(WideShared& s, double x) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave_sum[threadIdx.x >> 6] = x;
  __syncthreads();
  return (s.wave_sum[0] + s.wave_sum[1]) + (s.wave_sum[2] + s.wave_sum[3]);
}

// Sum of exp(x - top). A logarithm of it is asked for in fp32: exponentials in fp32 are off by less than 2^-22 of
// each that counts, a thread's sum of at most 32 by as much again, and so is the logarithm, in all below 2^-21.
template <typename M, int N>
__device__ double exp_sum(WideShared& s, const M& m, float top) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    sum += m.x[i] == top ? 1.0f : __builtin_amdgcn_exp2f((m.x[i] - top) * 1.44269504f);
  return sum_all(s, (double)sum);
}

constexpr int kPartUnit = 49;           // a part's weights against its own largest: 2^-49, at most 8192 of them

// Without filters: a part's weight against its largest logit.
template <bool BF16, bool VEC, int N>
__global__ __launch_bounds__(kWide) void weigh(SampleArgs a, Shape sh) {
  __shared__ WideShared s;
  const int row_at = (int)blockIdx.x / sh.l.parts, n = (int)blockIdx.x % sh.l.parts;
  Mine<BF16, VEC, N> m;
  m.load(row_of(a, row_at), n * sh.l.per, a.V);
  fill_table(s.table);
  const Params par(a, row_at);
  Part part = {};
  const float top = of_key(largest<decltype(m), N>(s, m, part));
  u64 sum = 0;
  if (!par.greedy() && top > -INFINITY) {
    const Weights w = {top, kLog2e / (double)par.t, kPartUnit, s.table};
#pragma unroll
    for (int i = 0; i < N; ++i) sum += w(m.x[i]);
    u64 before;
    uint32_t c;
    scan<kWide>(s.wave_mass, s.wave_count, sum, 0, before, c, part.kept);
  }
  if (a.logprobs && top > -INFINITY) part.sum = exp_sum<decltype(m), N>(s, m, top);
  if (threadIdx.x == 0) sh.parts(a, row_at)[n] = part;
}

// The row's largest logit and its first place from the parts; false where the row gives no token.
__device__ bool largest_of_parts(Shared& s, const Part* parts, int n, float t, uint32_t& top, int& first) {
  if (threadIdx.x == 0) s.key = 0, s.index = 0xFFFFFFFFu, s.flag = t != t;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    if (parts[i].bad) s.flag = 1;
    atomicMax(&s.key, parts[i].top);
  }
  __syncthreads();
  top = s.key;
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (parts[i].top == top) atomicMin(&s.index, (uint32_t)parts[i].at);
  __syncthreads();
  first = (int)s.index;
  return !s.flag && of_key(top) > -INFINITY;
}

__device__ void write_none(const SampleArgs& a, int row) {
  if (threadIdx.x == 0) {
    a.tokens[row] = -1;
    if (a.logprobs) a.logprobs[row] = kNaN;
  }
}
template <bool BF16>
__device__ void write_token(const SampleArgs& a, int row_at, int token, float top, const Part* parts, int n,
                            Shared& s) {
  if (a.logprobs) {                     // (a sum in a fixed order)
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float part = of_key(parts[i].top);
      if (part > -INFINITY)
        sum += parts[i].sum * (part == top ? 1.0 : exp2_64(((double)part - (double)top) * kLog2e, s.table));
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_mass[threadIdx.x >> 6] = (u64)__double_as_longlong(sum);
    __syncthreads();
    if (threadIdx.x == 0) {
      sum = 0.0;
      for (int i = 0; i < kThreads / 64; ++i) sum += __longlong_as_double((long long)s.wave_mass[i]);
      const float x = logit<BF16>(row_of(a, row_at), token);
      a.logprobs[row_at] = (float)((x == top ? 0.0 : (double)x - (double)top) - log(sum));
    }
  }
  if (threadIdx.x == 0) a.tokens[row_at] = token;
}

// The first place in [from, to) at which the cumulated weight exceeds target, in order of places: runs of
// consecutive elements a thread.
template <bool BF16, typename F>
__device__ int pass_at(Shared& s, const void* row, int from, int to, u64 target, const F& weight) {
  if (threadIdx.x == 0) s.found = -1;
  const int run = ceil_div(to - from, kThreads), i0 = from + (int)threadIdx.x * run, i1 = min(i0 + run, to);
  u64 mine = 0, before, all;
  uint32_t c;
  for (int i = i0; i < i1; ++i) mine += weight(logit<BF16>(row, i), i);
  scan(s, mine, 0, before, c, all);
  // (a target past the sum, by rounding, takes the last element of any weight)
  target = min(target, all - 1);
  if (before <= target && before + mine > target) {
    u64 sum = before;
    for (int i = i0; i < i1; ++i) {
      sum += weight(logit<BF16>(row, i), i);
      if (sum > target) {
        s.found = i;
        break;
      }
    }
  }
  __syncthreads();
  return s.found;
}

// The part in which the cumulated sum of weight_of(part) passes uniform times all of it: the part, and what is
// left of the target in it. Sums of the parts lie in s.tile_mass.
__device__ int part_of(Shared& s, int parts, float uniform, u64& target) {
  // runs of consecutive parts a thread
  if (threadIdx.x == 0) s.found = parts - 1, s.above_mass = 0;
  const int run = ceil_div(parts, kThreads), i0 = (int)threadIdx.x * run, i1 = min(i0 + run, parts);
  u64 mine = 0, before, Z;
  uint32_t c;
  for (int i = i0; i < i1; ++i) mine += s.tile_mass[i];
  scan(s, mine, 0, before, c, Z);
  const u64 all = target_of(uniform, Z);
  if (before <= all && before + mine > all) {
    u64 sum = before;
    for (int i = i0; i < i1; ++i) {
      if (sum + s.tile_mass[i] > all) {
        s.found = i, s.above_mass = all - sum;
        break;
      }
      sum += s.tile_mass[i];
    }
  }
  __syncthreads();
  target = s.above_mass;
  return s.found;
}

// Without filters: the token from the parts' weights.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void pick(SampleArgs a, Shape sh) {
  __shared__ Shared s;
  const int row_at = blockIdx.x, n = sh.l.parts;
  const Part* parts = sh.parts(a, row_at);
  const Params par(a, row_at);
  fill_table(s.table);
  uint32_t top_key;
  int token;
  if (!largest_of_parts(s, parts, n, par.t, top_key, token)) return write_none(a, row_at);
  const float top = of_key(top_key);
  if (!par.greedy()) {
    const double rate = kLog2e / (double)par.t, unit = ldexp(1.0, unit_shift(a.V) - kPartUnit);
    const auto factor = [&](int i) {
      const float x = of_key(parts[i].top);
      return x == -INFINITY ? 0.0 : x == top ? 1.0 : exp2_64(((double)x - (double)top) * rate, s.table);
    };
    for (int i = threadIdx.x; i < n; i += kThreads) s.tile_mass[i] = (u64)((double)parts[i].kept * factor(i) * unit + 0.5);
    __syncthreads();
    u64 target;
    const int at = part_of(s, n, a.uniform[row_at], target);
    const Weights w = {of_key(parts[at].top), rate, kPartUnit, s.table};
    // what is left of the target, in the part's own units
    const u64 inside = (u64)((double)target / (double)s.tile_mass[at] * (double)parts[at].kept);
    token = pass_at<BF16>(s, row_of(a, row_at), at * sh.l.per, min((at + 1) * sh.l.per, a.V), inside,
                          [&](float x, int) { return w(x); });
  }
  write_token<BF16>(a, row_at, token, top, parts, n, s);
}

// The largest value of a bin of keys (of finite ones).
__device__ __forceinline__ float bin_value(uint32_t bin) { return of_key(bin << kBinShift | ((1u << kBinShift) - 1)); }

template <bool BF16, bool VEC, int N>
__global__ __launch_bounds__(kWide) void survey(SampleArgs a, Shape sh) {
  __shared__ WideShared s;
  const int row_at = (int)blockIdx.x / sh.l.parts, n = (int)blockIdx.x % sh.l.parts, tid = threadIdx.x;
  Mine<BF16, VEC, N> m;
  m.load(row_of(a, row_at), n * sh.l.per, a.V);
  fill_table(s.table);
  const Params par(a, row_at);
  const bool bins = !par.greedy() && (par.by_k || par.by_p);
  if (bins)
    for (int i = tid; i < kBins; i += kWide) s.bins[i] = 0;
  Part part = {};
  const float top = of_key(largest<decltype(m), N>(s, m, part));
  if (bins) {
    // The bin of the part's largest logit, which may be the row's, counts against that logit: against the
    // bin's largest possible value it could be all but nothing. No other bin's value is above the row's largest.
    const double rate = kLog2e / (double)par.t;
    const uint32_t top_bin = part.top >> kBinShift;
    const Weights w = {top, rate, kPartUnit, s.table};
    u64 near = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!(m.x[i] > -INFINITY)) continue;
      const uint32_t bin = key_of(m.x[i]) >> kBinShift;
      u64 x = 0;
      if (par.by_p) {
        if (bin == top_bin) near += w(m.x[i]);
        else x = to_units(exp2_64(((double)m.x[i] - (double)bin_value(bin)) * rate, s.table, kRelative));
      }
      atomicAdd(&s.bins[bin], x << kCountBits | 1);
    }
    u64 before;
    uint32_t c;
    scan<kWide>(s.wave_mass, s.wave_count, near, 0, before, c, part.near);
    __syncthreads();
    RowSpace& row = sh.space(a, row_at);
    for (int i = tid; i < kBins; i += kWide) {
      const u64 x = s.bins[i];
      if (!x) continue;
      atomicAdd(&row.count[i], (uint32_t)(x & ((1u << kCountBits) - 1)));
      if (x >> kCountBits) atomicAdd(&row.mass[i], x >> kCountBits);
    }
  }
  if (a.logprobs && top > -INFINITY) part.sum = exp_sum<decltype(m), N>(s, m, top);
  if (tid == 0) sh.parts(a, row_at)[n] = part;
}

struct CollectShared : WideShared {
  uint32_t low, high;                   // keys of the listed bins: low <= key < high
  uint32_t elements, begin;
  u64 below, above_count, above_mass;
};

template <bool BF16, bool VEC, int N>
__global__ __launch_bounds__(kWide) void collect(SampleArgs a, Shape sh) {
  __shared__ CollectShared s;
  const int row_at = (int)blockIdx.x / sh.l.parts, n = (int)blockIdx.x % sh.l.parts, tid = threadIdx.x;
  const Params par(a, row_at);
  if (par.greedy()) return;
  Mine<BF16, VEC, N> m;
  m.load(row_of(a, row_at), n * sh.l.per, a.V);
  Part* parts = sh.parts(a, row_at);
  RowSpace& row = sh.space(a, row_at);
  fill_table(s.table);
  if (tid == 0) s.top = 0, s.bad = 0, s.low = s.high = 0, s.below = s.above_count = s.above_mass = 0;
  for (int i = tid; i < kBins; i += kWide) s.bins[i] = 0;
  __syncthreads();
  for (int i = tid; i < sh.l.parts; i += kWide) {
    atomicMax(&s.top, parts[i].top);
    if (parts[i].bad) s.bad = 1;
  }
  __syncthreads();
  const float top = of_key(s.top);
  if (s.bad || top == -INFINITY) return;
  const double rate = kLog2e / (double)par.t;
  const int shift = unit_shift(a.V);
  const Weights w = {top, rate, shift, s.table};
  bool by_k = false;
  if (par.by_k || par.by_p) {
    if (par.by_p) {
      for (int i = tid; i < sh.l.parts; i += kWide)
        if (parts[i].near)
          atomicAdd(&s.bins[parts[i].top >> kBinShift],
                    (u64)((double)parts[i].near * w.real(of_key(parts[i].top)) * ldexp(1.0, shift - kPartUnit) + 0.5));
      __syncthreads();
    }
    // bins from the highest, 8 a thread
    constexpr int kEach = kBins / kWide;
    u64 mass[kEach], mine = 0, before_m, all_m;
    uint32_t count[kEach], have = 0, before_c;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint32_t bin = kBins - 1 - kEach * tid - j;
      count[j] = row.count[bin], mass[j] = 0;
      if (par.by_p && count[j]) {
        mass[j] = s.bins[bin];
        const u64 x = row.mass[bin];    // (none in the bin of the row's largest)
        if (x) mass[j] += (u64)((double)x * w.real(bin_value(bin)) * ldexp(1.0, shift - kRelative) + 0.5);
      }
      have += count[j], mine += mass[j];
    }
    scan<kWide>(s.wave_mass, s.wave_count, mine, have, before_m, before_c, all_m);
    if (tid == kWide - 1) s.elements = before_c + have;
    __syncthreads();
    by_k = par.by_k && s.elements >= (uint32_t)par.k;
    // The bins to list: that of the cut by top-k; that by top-p; with both all from the highest in which the cut
    // by top-p can be (if nothing of top-k's bin counts) to top-k's.
    if (by_k) {
      u64 ac = before_c, am = before_m;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (ac < (u64)par.k && ac + count[j] >= (u64)par.k) {
          const uint32_t bin = kBins - 1 - kEach * tid - j;
          s.low = bin << kBinShift, s.high = (bin + 1) << kBinShift;
          s.above_count = ac, s.above_mass = am;
        }
        ac += count[j], am += mass[j];
      }
      __syncthreads();
    }
    if (par.by_p) {
      // (with top-k a little less: the bins' sums are rounded)
      const double want = ceil((double)par.p * (by_k ? (double)s.above_mass * (1.0 - 1e-9) : (double)all_m));
      const u64 target = (u64)fmax(want, 1.0);
      __syncthreads();
      u64 ac = before_c, am = before_m;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        if (am < target && am + mass[j] >= target) {
          const uint32_t bin = kBins - 1 - kEach * tid - j;
          s.high = (bin + 1) << kBinShift;
          if (!by_k) s.low = bin << kBinShift, s.below = all_m - am - mass[j];
          s.above_count = ac;
        }
        ac += count[j], am += mass[j];
      }
      __syncthreads();
    }
  }
  const uint32_t low = s.low, high = s.high;
  // Weight of what is above, and the list. (Below `skip` a weight is certainly below min-p: no exponential.)
  const float skip = par.mp > 0.0f
                         ? (float)((double)top + log2((double)par.mp) / rate * 1.0001) - 1e-6f * (1.0f + fabsf(top))
                         : -INFINITY;
  u64 sum = 0;
  uint32_t entries = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = m.x[i];
    if (!(x > -INFINITY)) continue;
    const uint32_t key = key_of(x);
    if (key < low) continue;
    if (key < high) {
      ++entries;
      continue;
    }
    if (x < skip) continue;
    sum += w.at_least(x, par.mp);
  }
  u64 before_m, all_m;
  uint32_t before_c;
  scan<kWide>(s.wave_mass, s.wave_count, sum, entries, before_m, before_c, all_m);
  if (tid == kWide - 1) {
    const uint32_t all = before_c + entries;
    s.begin = all ? atomicAdd(&row.listed, all) : 0;
  }
  __syncthreads();
  Entry* list = sh.list(a, row_at);
  uint32_t at = s.begin + before_c;
  if (entries)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = m.x[i];
      const uint32_t key = key_of(x);
      if (!(x > -INFINITY) || key < low || key >= high) continue;
      if (at < (uint32_t)sh.l.most) list[at] = {w(x), key, m.place(i)};
      ++at;
    }
  if (tid == 0) {
    parts[n].kept = all_m;
    if (n == 0) row.below = s.below, row.above_count = s.above_count, row.low = low, row.high = high,
                row.by_k = by_k;
  }
}

struct ListSource {
  const Entry* list;
  __device__ uint32_t key(int i) const { return list[i].key; }
  __device__ u64 weight(int i) const { return list[i].weight; }
};

// The place of the `ties`-th of the entries at `cut`, in order of places: 8 of its 24 bits at a time.
__device__ int last_tie(Shared& s, const Entry* list, int n, uint32_t cut, u64 ties) {
  uint32_t at = 0;
  u64 left = ties;
  for (int level = 0; level < 3; ++level) {
    const int shift = 16 - 8 * level;
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) s.count[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (list[i].key == cut && (level == 0 || (uint32_t)list[i].at >> (shift + 8) == at >> (shift + 8)))
        atomicAdd(&s.count[((uint32_t)list[i].at >> shift) & 255], 1u);
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 sum = 0;
      uint32_t d = 0;
      while (d < 255 && sum + s.count[d] < left) sum += s.count[d++];
      s.key = d, s.above_count = sum;
    }
    __syncthreads();
    at |= s.key << shift, left -= s.above_count;
  }
  return (int)at;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void choose(SampleArgs a, Shape sh) {
  __shared__ Shared s;
  const int row_at = blockIdx.x, n = sh.l.parts;
  const Part* parts = sh.parts(a, row_at);
  const RowSpace& row = sh.space(a, row_at);
  const Params par(a, row_at);
  fill_table(s.table);
  uint32_t top_key;
  int token;
  if (!largest_of_parts(s, parts, n, par.t, top_key, token)) return write_none(a, row_at);
  const float top = of_key(top_key);
  if (!par.greedy()) {
    const int listed = (int)row.listed;
    if (listed > sh.l.most) return whole_row<BF16>(a, row_at, s);
    const Weights w = {top, kLog2e / (double)par.t, unit_shift(a.V), s.table};
    const Entry* list = sh.list(a, row_at);
    const ListSource source = {list};
    if (threadIdx.x == 0) s.key = 0, s.above_count = s.above_mass = 0;
    u64 above = 0, in_list = 0, before;
    uint32_t c;
    {
      u64 mine = 0;
      for (int i = threadIdx.x; i < n; i += kThreads) mine += parts[i].kept, s.tile_mass[i] = parts[i].kept;
      scan(s, mine, 0, before, c, above);
      mine = 0;
      for (int i = threadIdx.x; i < listed; i += kThreads) mine += list[i].weight;
      scan(s, mine, 0, before, c, in_list);
    }
    // (Where min-p takes from what is above the list it takes all of the list, and the cuts do not matter.)
    // (the digit that the listed keys share, where they lie in one bin, is not looked at)
    const int level = row.high - row.low == 1u << kBinShift;
    uint32_t cut = 0;
    u64 ties = 0, total = above + in_list + row.below;
    bool whole = true;                  // all of the list is kept
    if (row.by_k) {
      u64 ac = row.above_count, am = above;
      cut = level ? row.low : 0;
      find_cut<false>(s, listed, source, (u64)par.k, cut, ac, am, level);
      ties = (u64)par.k - ac, whole = false;
      total = am + ties * w(of_key(cut));
    }
    bool none = false;                  // nothing of it is
    if (par.by_p) {
      const double want = ceil((double)par.p * (double)total);
      if (!(want >= 1.0)) {
        cut = top_key, ties = 1, whole = false;
      } else if ((u64)want <= above) {
        none = true;
      } else if ((u64)want <= above + in_list) {
        u64 ac = row.above_count, am = above;
        const u64 target = min((u64)want, total);
        cut = level ? row.low : 0;
        find_cut<true>(s, listed, source, target, cut, ac, am, level);
        const u64 each = max(w(of_key(cut)), 1ull);
        ties = (target - am + each - 1) / each, whole = false;
      }
    }
    // the first `ties` elements at the cut: the place of the last of them
    int last = 0x7FFFFFFF;
    if (!whole && !none) {
      u64 mine = 0, at_cut;
      for (int i = threadIdx.x; i < listed; i += kThreads) mine += list[i].key == cut;
      scan(s, mine, 0, before, c, at_cut);
      if (ties < at_cut) last = last_tie(s, list, listed, cut, ties);
    }
    const auto listed_kept = [&](uint32_t key, int at, u64 weight) -> u64 {
      if (none || (!whole && (key < cut || (key == cut && at > last)))) return 0;
      return par.mp > 0.0f && !(w.real(of_key(key)) >= (double)par.mp) ? 0 : weight;
    };
    __syncthreads();
    for (int i = threadIdx.x; i < listed; i += kThreads) {
      const u64 x = listed_kept(list[i].key, list[i].at, list[i].weight);
      if (x) atomicAdd(&s.tile_mass[list[i].at / sh.l.per], x);
    }
    __syncthreads();
    u64 target;
    const int at = part_of(s, n, a.uniform[row_at], target);
    // the listed bins again, to tell what is above them
    const uint32_t low = row.low, high = row.high;
    token = pass_at<BF16>(s, row_of(a, row_at), at * sh.l.per, min((at + 1) * sh.l.per, a.V), target,
                          [&](float x, int i) -> u64 {
                            const uint32_t key = key_of(x);
                            if (x == -INFINITY || key < low) return 0;
                            if (key < high) return listed_kept(key, i, w(x));
                            return w.at_least(x, par.mp);
                          });
  }
  write_token<BF16>(a, row_at, token, top, parts, n, s);
}

}  // namespace

bool sample_filters(const SampleArgs& a) {
  return a.top_k || a.top_p || a.min_p || (a.top_k_all >= 1 && a.top_k_all < a.V) || a.top_p_all < 1.0f ||
         a.min_p_all > 0.0f;
}

namespace {

template <bool BF16, bool VEC, int N>
void launch_wide(const SampleArgs& a, const Shape& sh, hipStream_t stream) {
  const unsigned grid = (unsigned)(a.rows * sh.l.parts);
  if (!sh.filters) {
    weigh<BF16, VEC, N><<<grid, kWide, 0, stream>>>(a, sh);
    pick<BF16><<<a.rows, kThreads, 0, stream>>>(a, sh);
    return;
  }
  clear_rows<<<a.rows, kWide, 0, stream>>>(a, sh);
  survey<BF16, VEC, N><<<grid, kWide, 0, stream>>>(a, sh);
  collect<BF16, VEC, N><<<grid, kWide, 0, stream>>>(a, sh);
  choose<BF16><<<a.rows, kThreads, 0, stream>>>(a, sh);
}
template <bool BF16>
void launch_wide(const SampleArgs& a, const Shape& sh, hipStream_t stream) {
  const bool vec = ((uintptr_t)a.logits | (size_t)(a.rows > 1 ? a.row_stride * (BF16 ? 2 : 4) : 0)) % 16 == 0;
  if (sh.l.per == 8192) vec ? launch_wide<BF16, true, 32>(a, sh, stream) : launch_wide<BF16, false, 32>(a, sh, stream);
  else vec ? launch_wide<BF16, true, 8>(a, sh, stream) : launch_wide<BF16, false, 8>(a, sh, stream);
}

// Vocabularies up to this take one workgroup a row.
constexpr int kSmall = 4096;

}  // namespace

long sample_workgroups(int rows, int V) { return V <= kSmall ? rows : (long)rows * layout_of(rows, V, false).parts; }

size_t sample_workspace(int rows, int V, bool filters) {
  return V <= kSmall ? 0 : rows * layout_of(rows, V, filters).row;
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  if (a.V <= kSmall) {
    if (a.bf16) sample_rows<true><<<a.rows, kThreads, 0, stream>>>(a);
    else sample_rows<false><<<a.rows, kThreads, 0, stream>>>(a);
  } else {
    const bool filters = sample_filters(a);
    const Shape sh = {layout_of(a.rows, a.V, filters), filters};
    if (a.bf16) launch_wide<true>(a, sh, stream);
    else launch_wide<false>(a, sh, stream);
  }
  return hipGetLastError();
}

}  // namespace dec
