// Per-head RMSNorm of queries and keys, the rotation, and the rounding of new keys and values into
// the 4-bit cache, for gfx950.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w,  (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
//
// One pass: each lane holds 8 channels of one token's head (16 bytes), D / 8 lanes a head, so a wave
// has 64 / (D / 8) consecutive tokens of one head. The pair partner of (p, p + rot / 2) is another
// lane's; its normed channels come over the lane permute network. A wave keeps its tokens' cosines and
// sines in registers and walks over several heads, the next one's 16 bytes a lane always in flight.
// Four consecutive tokens of a wave at D = 128 are one run of 256 bytes of the value layout where
// they fall on consecutive slots.
//
// Bounded by HBM: 4096 tokens of 48 query, 16 key and 16 value heads of 128 with their cache slots, 143
// MB, 34 us, 4.2 TB/s of the 5.1 that a large copy reaches (vector work alone would take half of it);
// 3777 tokens of 24 + 4 heads of 256, three axes: 111 MB, 26 us, 4.2 TB/s. Two or four heads in flight
// were no faster (fewer waves fit). One token: 4 us, the latency of three dependent reads.
//
// Every floating-point step is fixed (no contraction into fused multiply-adds), so the outputs and
// the cache's bytes are the same bits as a plain fp32 evaluation in this order: with keys rounded to
// 4 bits, a last-place difference would otherwise move a code by a whole step now and then.
#include "kv4_attn.h"
#include "kv4_internal.h"

namespace kv4 {
namespace {

#pragma clang fp contract(off)


__device__ __forceinline__ void unpack8(const uint4 r, float x[8]) {
  x[0] = bf16_lo(r.x), x[1] = bf16_hi(r.x), x[2] = bf16_lo(r.y), x[3] = bf16_hi(r.y);
  x[4] = bf16_lo(r.z), x[5] = bf16_hi(r.z), x[6] = bf16_lo(r.w), x[7] = bf16_hi(r.w);
}

__device__ __forceinline__ uint4 pack8(const float y[8]) {
  return make_uint4(bf16x2(y[0], y[1]), bf16x2(y[2], y[3]), bf16x2(y[4], y[5]),
                    bf16x2(y[6], y[7]));
}

// A position's row of the table, or -1.
__device__ __forceinline__ long table_row(const RopeArgs& a, int axis, int t) {
  if (axis < 0 || axis >= a.axes) return -1;
  const size_t at = (size_t)axis * a.pos_stride + t;
  const long p = a.flags & KV4_POS_I32 ? (long) reinterpret_cast<const int*>(a.pos)[at]
                                       : (long) reinterpret_cast<const int64_t*>(a.pos)[at];
  return p < a.rows ? p : -1;
}

// N consecutive entries of a row of the table; those of no row are NaN.
template <int N>
__device__ __forceinline__ void table_at(const RopeArgs& a, long row, int col, float out[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = __uint_as_float(0x7FC00000u);
  if (row < 0) return;
  const size_t at = (size_t)row * a.rot + col;
  if (a.flags & KV4_TABLE_BF16) {
    uint16_t x[N];
    __builtin_memcpy(x, reinterpret_cast<const uint16_t*>(a.table) + at, sizeof(x));
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = __uint_as_float((uint32_t)x[i] << 16);
  } else {
    __builtin_memcpy(out, reinterpret_cast<const float*>(a.table) + at, 4 * N);
  }
}

// Cosines and sines of N pairs from `pair` on, at token t.
template <int N>
__device__ __forceinline__ void turns_of(const RopeArgs& a, int pair, int t, float cs[N],
                                         float sn[N]) {
  const int half = a.rot >> 1;
  int axis[N] = {};
  bool one = true;                    // one axis for all of them
  if (a.axis) {
    __builtin_memcpy(axis, a.axis + pair, sizeof(axis));
#pragma unroll
    for (int i = 1; i < N; ++i) one = one && axis[i] == axis[0];
  }
  if (__ballot(!one) == 0) {
    const long row = table_row(a, axis[0], t);
    table_at<N>(a, row, pair, cs);
    table_at<N>(a, row, half + pair, sn);
    return;
  }
  long row[N];
#pragma unroll
  for (int i = 0; i < N; ++i) row[i] = table_row(a, axis[i], t);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    table_at<1>(a, row[i], pair + i, cs + i);
    table_at<1>(a, row[i], half + pair + i, sn + i);
  }
}

// The largest magnitude's bits over the 4 lanes of a block of 32 channels. Integer order is the
// magnitudes' order, with NaN above infinity.
__device__ __forceinline__ uint32_t block_amax(const float y[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(y[i]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 1));
  return max(m, (uint32_t)__shfl_xor((int)m, 2));
}

// 8 channels (lane j of the head) of a key or value as codes and scale into the token's places.
template <int D>
__device__ __forceinline__ void store_cached(uint8_t* group, int token, int j, const float y[8],
                                             bool value) {
  using G = Group<D>;
  const uint32_t e = scale_byte(block_amax(y));
  const uint32_t c = codes8(y, e);
  const int blk = j >> 2;
  if (!value) {
    *reinterpret_cast<uint32_t*>(group + G::kKeys + token * (D / 2) + 4 * j) = c;
    if ((j & 3) == 0) group[G::kKeyScales + token * (D / kBlock) + blk] = (uint8_t)e;
    return;
  }
  const int g = token >> 2, i = token & 3;
  if constexpr (G::kRun == 8) {
    const int plane = j >> 4, r = j & 15;
    *reinterpret_cast<uint32_t*>(group + G::kValues + (((plane * 4 + g) * 16 + r) * 4 + i) * 4) = c;
  } else {
    uint8_t* at = group + G::kValues + ((g * 16 + 2 * j) * 4 + i) * 2;
    *reinterpret_cast<uint16_t*>(at) = (uint16_t)c;
    *reinterpret_cast<uint16_t*>(at + 8) = (uint16_t)(c >> 16);
  }
  if ((j & 3) == 0) group[G::kValueScales + blk * kGroup + token] = (uint8_t)e;
}

// What a lane keeps: its place in the head, its token, and the token's turns.
template <int D>
struct Lane {
  static constexpr int kLanes = D / 8;          // lanes of a head
  static constexpr int kTokens = 64 / kLanes;   // tokens of a wave
  int j, t, partner;          // partner: lane of the other channels of its pairs
  bool live, turns;
  float cs[8], sn[8];         // of its channels; the sign of a pair's first is in its sine
  uint8_t* token_at;          // the token's page, or null
  int place;                  // and its place in there
};

enum Kind { kQuery, kKey, kValue };

// Heads [h0, h1) of the queries, the keys or the values.
template <int D, Kind K>
__device__ __forceinline__ void walk(const RopeArgs& a, const Lane<D>& l, int h0, int h1) {
  if (h0 >= h1) return;
  const Heads& src = K == kQuery ? a.q : K == kKey ? a.k : a.v;
  const int c0 = 8 * l.j;
  const uint16_t* from = src.p + (size_t)(l.live ? l.t : a.T - 1) * src.ts + c0;
  // The next head is asked for a head ahead of its use (past the end the last one again, a cache hit:
  // a load that is always issued lets the wait count those in flight).
  auto load = [&](int h) {
    return *reinterpret_cast<const uint4*>(from + (size_t)min(h, h1 - 1) * src.hs);
  };
  uint4 raw = load(h0);
  const uint16_t* weights = K == kQuery ? a.qw : K == kKey ? a.kw : nullptr;
  float w[8];
  if (weights) {
    unpack8(*reinterpret_cast<const uint4*>(weights + c0), w);
    if (a.flags & KV4_PLUS_ONE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = w[i] + 1.0f;
    }
  }
  const int groups = 1 << (a.page_shift - 4);
  for (int h = h0; h < h1; ++h) {
    float x[8];
    unpack8(raw, x);
    raw = load(h + 1);
    if (weights) {
      const float s0 = x[0] * x[0] + x[4] * x[4], s1 = x[1] * x[1] + x[5] * x[5];
      const float s2 = x[2] * x[2] + x[6] * x[6], s3 = x[3] * x[3] + x[7] * x[7];
      float s = (s0 + s2) + (s1 + s3);
#pragma unroll
      for (int m = Lane<D>::kLanes / 2; m > 0; m >>= 1) s = s + __shfl_xor(s, m);
      const float r = 1.0f / sqrtf(s * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
    }
    if (K != kValue && a.rot) {
      float y[8];
      if (a.flags & KV4_ADJACENT) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] * l.cs[i] + x[i ^ 1] * l.sn[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] * l.cs[i] + __shfl(x[i], l.partner) * l.sn[i];
      }
      if (l.turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i];
      }
    }
    if (K == kQuery || (K == kKey && !a.cache)) {
      uint16_t* out = K == kQuery ? a.q_out : a.k_out;
      const int H = K == kQuery ? a.Hq : a.Hkv;
      if (l.live) *reinterpret_cast<uint4*>(out + ((size_t)l.t * H + h) * D + c0) = pack8(x);
    } else if (l.token_at) {           // (all lanes of a head or none)
      store_cached<D>(l.token_at + (size_t)(h * groups + (l.place >> 4)) * Group<D>::kBytes,
                      l.place & 15, l.j, x, K == kValue);
    }
  }
}

// waves: [ceil(T / tokens of a wave)][head chunks]; a head index runs over the queries, the keys and
// (with a cache) the values.
template <int D>
__global__ __launch_bounds__(256) void rope_rows(RopeArgs a, int heads, int heads_per_wave,
                                                 int chunks, int waves) {
  const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (wave >= waves) return;             // whole waves leave
  const int lane = threadIdx.x & 63;
  const int h0 = (wave % chunks) * heads_per_wave;
  const int h1 = min(h0 + heads_per_wave, heads);
  Lane<D> l;
  l.j = lane & (Lane<D>::kLanes - 1);
  l.t = (wave / chunks) * Lane<D>::kTokens + lane / Lane<D>::kLanes;
  l.live = l.t < a.T;
  const int t = l.live ? l.t : a.T - 1;
  const int c0 = 8 * l.j, half = a.rot >> 1;
  l.turns = c0 < a.rot;
  l.partner = !l.turns ? lane : c0 < half ? lane + (half >> 3) : lane - (half >> 3);
#pragma unroll
  for (int i = 0; i < 8; ++i) l.cs[i] = 1.0f, l.sn[i] = 0.0f;
  if (l.turns && h0 < a.Hq + a.Hkv) {
    if (a.flags & KV4_ADJACENT) {
      float cs[4], sn[4];
      turns_of<4>(a, c0 >> 1, t, cs, sn);
#pragma unroll
      for (int i = 0; i < 8; ++i) l.cs[i] = cs[i >> 1], l.sn[i] = i & 1 ? sn[i >> 1] : -sn[i >> 1];
    } else {
      turns_of<8>(a, c0 < half ? c0 : c0 - half, t, l.cs, l.sn);
#pragma unroll
      for (int i = 0; i < 8; ++i) l.sn[i] = c0 < half ? -l.sn[i] : l.sn[i];
    }
  }
  l.token_at = nullptr, l.place = 0;
  if (a.cache && l.live) {
    const long slot = a.slots[t], page = slot >> a.page_shift;
    l.place = (int)(slot & ((1 << a.page_shift) - 1));
    if (slot >= 0 && page < a.pages) l.token_at = a.cache + (size_t)page * a.page_stride;
  }
  walk<D, kQuery>(a, l, h0, min(h1, a.Hq));
  walk<D, kKey>(a, l, max(h0 - a.Hq, 0), min(h1 - a.Hq, a.Hkv));
  walk<D, kValue>(a, l, max(h0 - a.Hq - a.Hkv, 0), h1 - a.Hq - a.Hkv);
}

template <int D>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
  constexpr int kTokens = Lane<D>::kTokens;
  const int heads = a.Hq + a.Hkv + (a.cache ? a.Hkv : 0);
  const int rows = ceil_div(a.T, kTokens);
  // A wave walks over several heads where that still leaves 16 waves a CU: their cosines and sines
  // are read once. (Up to 16 heads: 8 took 28.9 us in place of 27.0 at 3777 tokens of 28 heads of 256,
  // 32 the same.)
  const long most = (long)rows * heads / 4096;
  const int chunks = ceil_div(heads, most < 1 ? 1 : most > 16 ? 16 : (int)most);
  const int per = ceil_div(heads, chunks);
  const int waves = rows * chunks;
  rope_rows<D><<<ceil_div(waves, 4), 256, 0, stream>>>(a, heads, per, chunks, waves);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch<64>(a, stream) : d == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace kv4
