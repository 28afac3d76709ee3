// One token of each row of logits by temperature, top-k, top-p and min-p from a given uniform number, for
// gfx950.
//
// What top-k and top-p keep is a prefix of the row in descending order, ties by index: all elements above a
// cut key and the first few at it. The cut is found digit by digit of the 32-bit keys (11, 11 and 10 bits),
// from histograms of how many elements, and of how much weight, have each digit after the digits found so
// far. Weights are exp in 64 bits, added as integers of 2^-s: the sums are exact and the same in any order,
// which the atomics of a histogram need, and with s = 62 - ceil(log2 V) a row's sum is off by no more than
// 2^-(s + 1) an element, 3e-12 of the largest weight in all for V = 131072 in the mean.
#include "decode_ops.h"
#include "dec_internal.h"

namespace dec {
namespace {

constexpr int kThreads = 1024, kBins = 2048, kTile = 4096, kMaxTiles = 4096;
typedef unsigned long long u64;

// Order-preserving bits of a float that is not NaN; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct Weights {
  float top;
  double inverse_t, unit;               // 1 / t, 2^s
  __device__ double real(float x) const {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inverse_t);
  }
  __device__ u64 operator()(float x) const { return x == -INFINITY ? 0 : (u64)__double2ull_rn(real(x) * unit); }
};

struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 wave_mass[16];
  uint32_t wave_count[16];
  u64 tile_mass[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  uint32_t key, index;
  u64 above_count, above_mass;
  int flag, found;
};

// Sums of the threads before this one, and of all.
__device__ void scan(Shared& s, u64 m, uint32_t c, u64& before_m, uint32_t& before_c, u64& all_m) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 im = m;
  uint32_t ic = c;
  for (int d = 1; d < 64; d <<= 1) {
    const u64 pm = __shfl_up(im, d);
    const uint32_t pc = __shfl_up(ic, d);
    if (lane >= d) im += pm, ic += pc;
  }
  __syncthreads();
  if (lane == 63) s.wave_mass[wave] = im, s.wave_count[wave] = ic;
  __syncthreads();
  before_m = im - m, before_c = ic - c, all_m = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before_m += s.wave_mass[w], before_c += s.wave_count[w];
    all_m += s.wave_mass[w];
  }
}

template <bool BF16>
__device__ __forceinline__ float logit(const void* row, int i) {
  return BF16 ? bf16_f32(((const uint16_t*)row)[i]) : ((const float*)row)[i];
}

// The cut at which the prefix of the order has `target` elements (BY_MASS: that much weight, > 0): its key,
// and what lies above the key.
template <bool BF16, bool BY_MASS>
__device__ void find_cut(Shared& s, const void* row, int V, const Weights& w, u64 target, uint32_t& key,
                         u64& above_count, u64& above_mass) {
  const int tid = threadIdx.x;
  key = 0, above_count = above_mass = 0;
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
    const uint32_t fixed = level == 0 ? 0u : ~0u << (shift + bits);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    for (int i = tid; i < V; i += kThreads) {
      const float x = logit<BF16>(row, i);
      const uint32_t k = key_of(x);
      if ((k & fixed) != key) continue;
      const uint32_t bin = (k >> shift) & ((1u << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], w(x));
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
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a) {
  __shared__ Shared s;
  const int row_at = blockIdx.x, tid = threadIdx.x, V = a.V;
  const void* row = (const char*)a.logits + (size_t)row_at * a.row_stride * (BF16 ? 2 : 4);
  const float t = a.temperature ? a.temperature[row_at] : a.temperature_all;
  const int k = a.top_k ? a.top_k[row_at] : a.top_k_all;
  const float p = a.top_p ? a.top_p[row_at] : a.top_p_all;
  const float mp = a.min_p ? a.min_p[row_at] : a.min_p_all;
  int shift = 62;
  while (shift > 0 && (1L << (62 - shift)) < V) --shift;

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
  Weights w = {of_key(s.key), 1.0 / (double)t, ldexp(1.0, shift)};
  const int first = (int)s.index;
  const bool none = s.flag || w.top == -INFINITY;
  if (none) {
    if (tid == 0) {
      a.tokens[row_at] = -1;
      if (a.logprobs) a.logprobs[row_at] = __uint_as_float(0x7FC00000u);
    }
    return;
  }
  int token = first;
  if (t > 0.0f && !(mp > 1.0f)) {
    uint32_t cut = 0;                   // kept: keys above it, and the first `ties` at it
    u64 ties = 0, above_count, above_mass;
    const bool by_k = k >= 1 && k < V, by_p = p < 1.0f;
    u64 total = 0;
    if (by_k) {
      find_cut<BF16, false>(s, row, V, w, (u64)k, cut, above_count, above_mass);
      ties = (u64)k - above_count;
      total = above_mass + ties * w(of_key(cut));
    }
    if (by_p) {
      if (!by_k) {
        u64 mine = 0, before;
        uint32_t c;
        for (int i = tid; i < V; i += kThreads) mine += w(logit<BF16>(row, i));
        scan(s, mine, 0, before, c, total);
      }
      const double want = ceil((double)p * (double)total);
      if (want >= 1.0) {
        const u64 target = min((u64)want, total);
        find_cut<BF16, true>(s, row, V, w, target, cut, above_count, above_mass);
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
      if (key < cut || (mp > 0.0f && !(w.real(x) >= (double)mp))) return 0;
      return w(x);
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
    // (a cumulated sum exceeds u Z, a whole number, where it exceeds what lies below u Z)
    u64 Z = 0, left = ties;
    for (int n = 0; n < tiles; ++n) {
      const u64 here = min((u64)s.tile_ties[n], left);
      Z += s.tile_mass[n] + here * each, left -= here;
    }
    const float u = fminf(fmaxf(a.uniform[row_at], 0.0f), 1.0f);
    const u64 target = min((u64)((double)u * (double)Z), Z - 1);
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
    const Weights one = {w.top, 1.0, w.unit};
    u64 mine = 0, before, total;
    uint32_t c;
    for (int i = tid; i < V; i += kThreads) mine += one(logit<BF16>(row, i));
    scan(s, mine, 0, before, c, total);
    if (tid == 0) {
      const float x = logit<BF16>(row, token);
      a.logprobs[row_at] =
          (float)((x == w.top ? 0.0 : (double)x - (double)w.top) - log((double)total / w.unit));
    }
  }
  if (tid == 0) a.tokens[row_at] = token;
}

}  // namespace

size_t sample_workspace(int, int, bool) { return 0; }

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  if (a.bf16) sample_rows<true><<<a.rows, kThreads, 0, stream>>>(a);
  else sample_rows<false><<<a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace dec
