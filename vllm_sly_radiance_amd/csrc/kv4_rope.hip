// Per-head RMSNorm of queries and keys, the rotation, and the rounding of new keys and values into
// the 4-bit cache, for gfx950.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w,  (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
//
// One pass: each lane holds 8 channels of one token's head (16 bytes), D / 8 lanes a head, so a wave
// has 64 / (D / 8) consecutive tokens of one head. The pair partner of (p, p + rot / 2) is another
// lane's; its 16 raw bytes come over the lane permute network, and its norm factor is the same.
// A wave keeps its tokens' cosines and sines in registers and walks over `heads_per_wave` heads.
// Four consecutive tokens of a wave at D = 128 are one run of 256 bytes of the value layout where
// they fall on consecutive slots.
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

__device__ __forceinline__ void weight8(const uint16_t* w, int c, bool plus_one, float out[8]) {
  unpack8(*reinterpret_cast<const uint4*>(w + c), out);
  if (plus_one) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = out[i] + 1.0f;
  }
}

__device__ __forceinline__ float table_at(const RopeArgs& a, long row, int col) {
  if (row < 0 || row >= a.rows) return __uint_as_float(0x7FC00000u);
  const size_t at = (size_t)row * a.rot + col;
  if (a.flags & KV4_TABLE_BF16)
    return __uint_as_float((uint32_t) reinterpret_cast<const uint16_t*>(a.table)[at] << 16);
  return reinterpret_cast<const float*>(a.table)[at];
}

__device__ __forceinline__ long position(const RopeArgs& a, int axis, int t) {
  if (axis < 0 || axis >= a.axes) return -1;
  const size_t at = (size_t)axis * a.pos_stride + t;
  return a.flags & KV4_POS_I32 ? (long) reinterpret_cast<const int*>(a.pos)[at]
                               : (long) reinterpret_cast<const int64_t*>(a.pos)[at];
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

// waves: [ceil(T / TPW)][head chunks]; a head index runs over the queries, the keys and (with a
// cache) the values.
template <int D>
__global__ __launch_bounds__(256) void rope_rows(RopeArgs a, int heads, int heads_per_wave,
                                                 int chunks, int waves) {
  using G = Group<D>;
  constexpr int kLanes = D / 8;          // lanes of a head
  constexpr int kTokens = 64 / kLanes;   // tokens of a wave
  const int wave = blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (wave >= waves) return;             // whole waves leave
  const int lane = threadIdx.x & 63;
  const int j = lane & (kLanes - 1);
  const int t = (wave / chunks) * kTokens + lane / kLanes;
  const bool live = t < a.T;
  const int tc = live ? t : a.T - 1;
  const int h0 = (wave % chunks) * heads_per_wave;
  const int h1 = min(h0 + heads_per_wave, heads);
  const int c0 = 8 * j;
  const int half = a.rot >> 1;
  const bool adjacent = a.flags & KV4_ADJACENT;
  const bool plus_one = a.flags & KV4_PLUS_ONE;
  const bool turns = c0 < a.rot;
  // lane of the partner channels (half style); a lane that does not rotate names itself
  const int partner =
      !turns || adjacent ? lane : c0 < half ? lane + (half >> 3) : lane - (half >> 3);
  const float sign = c0 < half ? -1.0f : 1.0f;

  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
  if (turns && h0 < a.Hq + a.Hkv) {
    if (!a.axis) {
      const long p = position(a, 0, tc);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = adjacent ? (c0 + i) >> 1 : (c0 < half ? c0 : c0 - half) + i;
        cs[i] = table_at(a, p, pair);
        sn[i] = table_at(a, p, half + pair);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = adjacent ? (c0 + i) >> 1 : (c0 < half ? c0 : c0 - half) + i;
        const long p = position(a, a.axis[pair], tc);
        cs[i] = table_at(a, p, pair);
        sn[i] = table_at(a, p, half + pair);
      }
    }
  }
  long slot = -1;
  uint8_t* page_at = nullptr;
  int place = 0;
  if (a.cache && live) {
    slot = a.slots[t];
    const long page = slot >> a.page_shift;
    place = (int)(slot & ((1 << a.page_shift) - 1));
    if (slot < 0 || page >= a.pages) slot = -1;
    else page_at = a.cache + (size_t)page * a.page_stride;
  }
  const int groups = 1 << (a.page_shift - 4);

  for (int h = h0; h < h1; ++h) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    const int hh = is_q ? h : is_v ? h - a.Hq - a.Hkv : h - a.Hq;
    const Heads& src = is_q ? a.q : is_v ? a.v : a.k;
    const uint4 raw =
        *reinterpret_cast<const uint4*>(src.p + (long)tc * src.ts + (long)hh * src.hs + c0);
    float x[8], y[8];
    unpack8(raw, x);
    if (is_v) {
      // amax goes over lanes: all of them take part
      if (page_at)
        store_cached<D>(page_at + (size_t)(hh * groups + (place >> 4)) * G::kBytes, place & 15, j,
                        x, true);
      continue;
    }
    const uint16_t* w = is_q ? a.qw : a.kw;
    float r = 1.0f;
    if (w) {
      const float s0 = x[0] * x[0] + x[4] * x[4], s1 = x[1] * x[1] + x[5] * x[5];
      const float s2 = x[2] * x[2] + x[6] * x[6], s3 = x[3] * x[3] + x[7] * x[7];
      float s = (s0 + s2) + (s1 + s3);
#pragma unroll
      for (int m = kLanes / 2; m > 0; m >>= 1) s = s + __shfl_xor(s, m);
      r = 1.0f / sqrtf(s * (1.0f / D) + a.eps);
      float wv[8];
      weight8(w, c0, plus_one, wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
    }
    if (a.rot) {
      if (adjacent) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          y[i] = x[i] * cs[i] - x[i + 1] * sn[i];
          y[i + 1] = x[i + 1] * cs[i] + x[i] * sn[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl(x[i], partner);
          y[i] = x[i] * cs[i] + sign * (other * sn[i]);
        }
      }
    }
    if (!turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
    }
    if (is_q || !a.cache) {
      uint16_t* out = is_q ? a.q_out : a.k_out;
      const int H = is_q ? a.Hq : a.Hkv;
      if (live)
        *reinterpret_cast<uint4*>(out + ((size_t)t * H + hh) * D + c0) = pack8(y);
    } else if (page_at) {
      store_cached<D>(page_at + (size_t)(hh * groups + (place >> 4)) * G::kBytes, place & 15, j, y,
                      false);
    }
  }
}

template <int D>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
  constexpr int kTokens = 64 / (D / 8);
  const int heads = a.Hq + a.Hkv + (a.cache ? a.Hkv : 0);
  const int rows = ceil_div(a.T, kTokens);
  // A wave walks over several heads where that still leaves 16 waves a CU: their cosines and sines
  // are read once.
  int per = (int)((long)rows * heads / 4096);
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  const int chunks = ceil_div(heads, per);
  const int waves = rows * chunks;
  rope_rows<D><<<ceil_div(waves, 4), 256, 0, stream>>>(a, heads, per, chunks, waves);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch<64>(a, stream) : d == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace kv4
