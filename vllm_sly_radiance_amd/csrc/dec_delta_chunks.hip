// The gated delta rule in chunks of 64 tokens, for gfx950: the form for prompts.
//
// With G the running sum of g in a chunk, S the state before it, and k, q of unit length, the tokens' u and
// outputs are (rows are tokens)
//   (1 + A) U = diag(beta) (V - diag(e^G) K S),   A_ij = beta_i e^(G_i - G_j) k_i . k_j for j < i
//   O = scale (diag(e^G) Q S + P U),              P_ij = e^(G_i - G_j) q_i . k_j for j <= i
//   S <- e^(G_63) S + K^T diag(e^(G_63 - G)) U
// A and P do not depend on the state: delta_prepare makes (1 + A)^-1 diag(beta), P and K^T of every chunk and
// head at once, and delta_chunks goes through a sequence's chunks with the state in registers.
//
// delta_chunks: a wave has 16 columns of a state, which do not meet others, so that its products need no
// other wave. As a matrix instruction's result a column is a lane and 4 rows of 16 lie in a lane's registers;
// as its operand a column is a lane and 8 of the 32 terms lie in them. The sums run over whatever order of
// terms both operands have, so with rows 8 g + 4 e + r of 32 in tile e, lane group g and register r, two
// result tiles are one operand as they are: S, X = V - K S and U go from product to product without
// leaving their lanes. The other operands are rows of 8 consecutive elements in memory.
//
// The operands that come from sums are in fp32 and a bf16 operand holds 8 bits: they are split into parts
// that add up to them, K and Q are exact.
#include "decode_ops.h"
#include "dec_delta.h"
#include "dec_internal.h"

namespace dec {
namespace {

constexpr int C = kChunk;
constexpr int kTParts = 3, kPParts = 2, kSParts = 3, kXParts = 3, kUParts = 2, kQParts = 2;
constexpr int kPad = 68;                // floats of a row of a chunk's matrices in LDS

// A chunk and head's part of the workspace.
struct ChunkHead {
  uint16_t t[kTParts][C][C];
  uint16_t p[kPParts][C][C];
  float k_factor[C], q_factor[C], u_factor[C];   // e^G / |k|, scale e^G / |q|, e^(G_63 - G) / |k|
  float decay, pad[3];                           // e^(G_63)
};

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v8bf load8(const uint16_t* p) { return *reinterpret_cast<const v8bf*>(p); }

// Parts of 8 fp32 values, each the rounding of what the ones before it leave.
template <int N>
__device__ __forceinline__ void split(const float x[8], v8bf part[N]) {
  uint32_t u[N][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo = x[2 * i], hi = x[2 * i + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      u[n][i] = bf16x2(lo, hi);
      if (n + 1 < N) lo -= bf16_lo(u[n][i]), hi -= bf16_hi(u[n][i]);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) part[n] = __builtin_bit_cast(v8bf, v4i{(int)u[n][0], (int)u[n][1], (int)u[n][2], (int)u[n][3]});
}

// K^T of a chunk and key head, [DK][C] bf16.
__device__ __forceinline__ uint16_t* delta_kt(const DeltaArgs& a, int dk, int c, int hk) {
  return (uint16_t*)((char*)a.workspace + a.kt) + ((size_t)c * a.Hk + hk) * dk * C;
}

// Chunk slots: sequence b's begin at starts[b] / 64 + b, so that total / 64 + batch slots hold all.
__device__ __forceinline__ int first_chunk(const Sequences& s, int b) {
  return min(max(s.starts[b], 0), s.total) / C + b;
}

// The sequence that chunk slot c belongs to: the last whose slots begin at it or before; -1 for none.
__device__ __forceinline__ int sequence_of(const Sequences& s, int c) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    const int b = b0 + lane;
    const int m = __popcll(__ballot(b < s.batch && first_chunk(s, min(b, s.batch - 1)) <= c));
    count += m;
    if (m < 64) break;
  }
  return count - 1;
}

__device__ __forceinline__ float sum_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <int DK>
struct PrepareShared {
  float a[C][kPad], t[C][kPad], p[C][kPad];
  float g_hi[C], g_lo[C], beta[C], rk[C], rq[C];
};

// One workgroup makes one chunk's matrices for one value head; wave w has rows 16 w .. 16 w + 15.
template <int DK>
__global__ __launch_bounds__(256) void delta_prepare(DeltaArgs a) {
  __shared__ __attribute__((aligned(16))) PrepareShared<DK> s;
  const int c = a.by_heads((int)blockIdx.x), h = (int)blockIdx.x - c * a.Hv;
  const int hk = a.by_group(h);
  const int b = sequence_of(a.s, c);
  if (b < 0) return;
  int first, n;
  rows_of(a.s, b, first, n);
  const int i0 = (c - first_chunk(a.s, b)) * C;
  if (i0 >= n) return;
  const int m = min(n - i0, C);
  const size_t row0 = (size_t)first + i0;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;

  constexpr int kSteps = DK / 32;
  const auto load = [&](const uint16_t* p, long ts, long hs, int tile, int step) {
    return load8(p + (row0 + min(16 * tile + col, m - 1)) * ts + hk * hs + 32 * step + 8 * g);
  };
  v8bf kf[kSteps], qf[kSteps];
  float kk = 0.0f, qq = 0.0f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    kf[i] = load(a.k, a.k_ts, a.k_hs, w, i), qf[i] = load(a.q, a.q_ts, a.q_hs, w, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) kk = fmaf((float)kf[i][j], (float)kf[i][j], kk), qq = fmaf((float)qf[i][j], (float)qf[i][j], qq);
  }
  kk = sum_groups(kk), qq = sum_groups(qq);
  if (g == 0) s.rk[16 * w + col] = 1.0f / sqrtf(kk + a.eps), s.rq[16 * w + col] = a.scale / sqrtf(qq + a.eps);
  if (w == 0) {
    // (decays below e^-200 are 0 either way; held to that, the sums stay finite)
    double sum = 0.0;
    float beta = 0.0f;
    if (lane < m) {
      const float x = log_decay(bf16_f32(a.a[(row0 + lane) * a.a_ts + h]), decay_rate(a.a_log[h]), a.dt_bias[h]);
      sum = x < -200.0f ? -200.0f : x;
      beta = sigmoid(bf16_f32(a.b[(row0 + lane) * a.b_ts + h]));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(sum, d);
      if (lane >= d) sum += y;
    }
    // two floats: differences of nearby sums keep the bits of what lies between them
    s.g_hi[lane] = (float)sum, s.g_lo[lane] = (float)(sum - (double)(float)sum), s.beta[lane] = beta;
  }
  __syncthreads();
  {
    const v4f rk = *(const v4f*)&s.rk[16 * w + 4 * g], rq = *(const v4f*)&s.rq[16 * w + 4 * g];
    const v4f hi = *(const v4f*)&s.g_hi[16 * w + 4 * g], lo = *(const v4f*)&s.g_lo[16 * w + 4 * g];
    const v4f beta = *(const v4f*)&s.beta[16 * w + 4 * g];
    for (int tile = 0; tile <= (w | 1); ++tile) {
      v4f ak = {}, aq = {};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const v8bf f = load(a.k, a.k_ts, a.k_hs, tile, i);
        ak = mfma(kf[i], f, ak), aq = mfma(qf[i], f, aq);
      }
      const int j = 16 * tile + col;
      const float rkj = s.rk[j], hj = s.g_hi[j], lj = s.g_lo[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * w + 4 * g + r;
        const float d = j <= i ? expf((hi[r] - hj) + (lo[r] - lj)) * rkj : 0.0f;
        s.a[i][j] = j < i ? beta[r] * d * rk[r] * ak[r] : 0.0f;
        s.p[i][j] = j <= i ? d * rq[r] * aq[r] : 0.0f;
      }
    }
  }
  __syncthreads();
  {
    // the inverse of a block on the diagonal, a column a lane
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x[4] = {i == col ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const v4f y = *(const v4f*)&s.a[16 * w + i][16 * w + j];
#pragma unroll
        for (int l = 0; l < 4; ++l)
          if (j + l < i) x[l] = fmaf(-y[l], t[j + l], x[l]);
      }
      t[i] = (x[0] + x[1]) + (x[2] + x[3]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (g == i >> 2) {
        s.t[16 * w + i][16 * w + col] = t[i];
        if (!(w & 1)) s.t[16 * w + i][16 * w + 16 + col] = 0.0f;
      }
  }
  __syncthreads();
  {
    // column block w of the inverse below the diagonal: T_iw = -T_ii sum_k A_ik T_kw
    v4f t[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[0][r] = s.t[16 * w + 4 * g + r][16 * w + col];
#pragma unroll
    for (int i = 1; i < 4; ++i) {       // block w + i
      if (w + i >= 4) break;
      v4f x = {};
#pragma unroll
      for (int k = 0; k < i; ++k) {
        const v4f y = *(const v4f*)&s.a[16 * (w + i) + col][16 * (w + k) + 4 * g];
#pragma unroll
        for (int r = 0; r < 4; ++r) x = __builtin_amdgcn_mfma_f32_16x16x4f32(y[r], t[k][r], x, 0, 0, 0);
      }
      const v4f y = *(const v4f*)&s.t[16 * (w + i) + col][16 * (w + i) + 4 * g];
      t[i] = v4f{};
#pragma unroll
      for (int r = 0; r < 4; ++r) t[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-y[r], x[r], t[i], 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) s.t[16 * (w + i) + 4 * g + r][16 * w + col] = t[i][r];
    }
  }
  __syncthreads();
  ChunkHead& out = ((ChunkHead*)a.workspace)[(size_t)c * a.Hv + h];
  const int i = tid >> 2;
  if (i >= 32 || (tid & 3) < 2)         // (the blocks that delta_chunks reads)
#pragma unroll
    for (int j0 = 0; j0 < 16; j0 += 8) {
      const int j = (tid & 3) * 16 + j0;
      float x[8], y[8];
#pragma unroll
      for (int l = 0; l < 8; ++l) x[l] = s.t[i][j + l] * s.beta[j + l], y[l] = s.p[i][j + l];
      v8bf tp[kTParts], pp[kPParts];
      split<kTParts>(x, tp), split<kPParts>(y, pp);
#pragma unroll
      for (int l = 0; l < kTParts; ++l) *(v8bf*)&out.t[l][i][j] = tp[l];
#pragma unroll
      for (int l = 0; l < kPParts; ++l) *(v8bf*)&out.p[l][i][j] = pp[l];
    }
  if (w == 0) {
    const float hi = s.g_hi[lane], lo = s.g_lo[lane], last = s.g_hi[C - 1], rest = s.g_lo[C - 1];
    const float in = expf(hi), there = lane < m ? 1.0f : 0.0f;
    out.k_factor[lane] = there * (in * s.rk[lane]);
    out.q_factor[lane] = in * s.rq[lane];
    out.u_factor[lane] = there * (expf((last - hi) + (rest - lo)) * s.rk[lane]);
    if (lane == 0) out.decay = expf(last);
  }
  if (hk * (a.Hv / a.Hk) == h) {        // K^T once for the heads that share it
    __syncthreads();
    uint16_t(*kt)[C + 8] = (uint16_t(*)[C + 8]) s.a;       // [DK][C], over a and t
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const v4i k = __builtin_bit_cast(v4i, kf[step]);
#pragma unroll
      for (int l = 0; l < 8; ++l) kt[32 * step + 8 * g + l][16 * w + col] = (uint16_t)((uint32_t)k[l / 2] >> (16 * (l & 1)));
    }
    __syncthreads();
    uint16_t* to = delta_kt(a, DK, c, hk);
    for (int x = tid; x < DK * C / 8; x += 256)
      *(v8bf*)(to + 8 * x) = *(const v8bf*)&kt[x / (C / 8)][x % (C / 8) * 8];
  }
}

// Token (or key channel) of row m of a tile: the order that makes two result tiles an operand.
__device__ __forceinline__ int place(int tile, int m) { return 32 * (tile >> 1) + 8 * (m >> 2) + 4 * (tile & 1) + (m & 3); }

template <int DK>
__global__ __launch_bounds__(256) void delta_chunks(DeltaArgs a, int dv) {
  constexpr int kSteps = DK / 32, kTiles = DK / 16;
  const int blocks = dv / 64;
  const int bh = (int)blockIdx.x / blocks;
  const int b = a.by_heads(bh), h = bh - b * a.Hv, hk = a.by_group(h);
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int col0 = ((int)blockIdx.x % blocks) * 64 + (threadIdx.x >> 6) * 16;
  int first, n;
  rows_of(a.s, b, first, n);
  const int c0 = first_chunk(a.s, b);

  v4f S[kTiles];
  const int read = a.s.read[b], write = a.s.write[b * a.s.write_stride];
  const size_t at = (size_t)h * DK * dv + col0 + col;
  const float fill = read < 0 ? 0.0f : __uint_as_float(0x7FC00000u);
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[j][r] = read >= 0 && read < a.s.slots
                    ? a.state[read * a.s.slot_stride + at + (size_t)place(j, 4 * g + r) * dv]
                    : fill;

  for (int i0 = 0; i0 < n; i0 += C) {
    const int m = min(n - i0, C);
    const size_t row0 = (size_t)first + i0;
    const ChunkHead& ch = ((const ChunkHead*)a.workspace)[(size_t)(c0 + i0 / C) * a.Hv + h];
    const uint16_t* kt = delta_kt(a, DK, c0 + i0 / C, hk);
    v4f x[4] = {}, o[4] = {};
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      v8bf sp[kSParts];
      const float y[8] = {S[2 * step][0],     S[2 * step][1],     S[2 * step][2],     S[2 * step][3],
                          S[2 * step + 1][0], S[2 * step + 1][1], S[2 * step + 1][2], S[2 * step + 1][3]};
      split<kSParts>(y, sp);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const size_t row = row0 + min(place(t, col), m - 1);
        const v8bf kf = load8(a.k + row * a.k_ts + hk * a.k_hs + 32 * step + 8 * g);
        const v8bf qf = load8(a.q + row * a.q_ts + hk * a.q_hs + 32 * step + 8 * g);
#pragma unroll
        for (int p = kSParts - 1; p >= 0; --p) x[t] = mfma(kf, sp[p], x[t]);
#pragma unroll
        for (int p = kQParts - 1; p >= 0; --p) o[t] = mfma(sp[p], qf, o[t]);
      }
    }
    v8bf xp[2][kXParts];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const v4f f = *(const v4f*)&ch.k_factor[32 * k + 8 * g + 4 * e];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = 32 * k + 8 * g + 4 * e + r;
          const float v = bf16_f32(a.v[(row0 + min(token, m - 1)) * a.v_ts + h * a.v_hs + col0 + col]);
          y[4 * e + r] = (token < m ? v : 0.0f) - f[r] * x[2 * k + e][r];
        }
      }
      split<kXParts>(y, xp[k]);
    }
    v4f u[4] = {};
    float bad = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int k = 0; k <= t / 2; ++k) {
        v8bf tf[kTParts];
#pragma unroll
        for (int p = 0; p < kTParts; ++p) tf[p] = load8(&ch.t[p][place(t, col)][32 * k + 8 * g]);
#pragma unroll
        for (int sum = (kTParts > kXParts ? kTParts : kXParts) - 1; sum >= 0; --sum)    // small products first
#pragma unroll
          for (int p = 0; p <= sum; ++p)
            if (p < kTParts && sum - p < kXParts) u[t] = mfma(tf[p], xp[k][sum - p], u[t]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) bad = fmaf(u[t][r], 0.0f, bad);
    }
    if (__any(bad != bad)) {
      // Something is not finite: token after token, so that no token sees a later one through a product
      // with zero.
      const float rate = decay_rate(a.a_log[h]), dt = a.dt_bias[h];
      for (int t = 0; t < m; ++t) {
        const size_t row = row0 + t;
        const float alpha = expf(log_decay(bf16_f32(a.a[row * a.a_ts + h]), rate, dt));
        const float beta = sigmoid(bf16_f32(a.b[row * a.b_ts + h]));
        const float v = bf16_f32(a.v[row * a.v_ts + h * a.v_hs + col0 + col]);
        float kk = 0.0f, qq = 0.0f, sk = 0.0f, sq = 0.0f;
        v8bf kf[kSteps], qf[kSteps];
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
          kf[step] = load8(a.k + row * a.k_ts + hk * a.k_hs + 32 * step + 8 * g);
          qf[step] = load8(a.q + row * a.q_ts + hk * a.q_hs + 32 * step + 8 * g);
#pragma unroll
          for (int l = 0; l < 8; ++l) {
            const float k = (float)kf[step][l], q = (float)qf[step][l];
            kk = fmaf(k, k, kk), qq = fmaf(q, q, qq), sk = fmaf(S[2 * step + l / 4][l & 3], k, sk);
          }
        }
        kk = sum_groups(kk), qq = sum_groups(qq), sk = sum_groups(sk);
        const float rk = 1.0f / sqrtf(kk + a.eps), rq = a.scale / sqrtf(qq + a.eps);
        const float ut = beta * (v - alpha * rk * sk) * rk;
#pragma unroll
        for (int step = 0; step < kSteps; ++step)
#pragma unroll
          for (int l = 0; l < 8; ++l) {
            const float y = fmaf((float)kf[step][l], ut, alpha * S[2 * step + l / 4][l & 3]);
            S[2 * step + l / 4][l & 3] = y;
            sq = fmaf(y, (float)qf[step][l], sq);
          }
        sq = rq * sum_groups(sq);
        if (g == 0) a.out[(row * a.Hv + h) * dv + col0 + col] = (uint16_t)bf16x2(sq, sq);
      }
      continue;
    }
    v8bf up[2][kUParts], sp[2][kSParts];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8], z[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const v4f f = *(const v4f*)&ch.u_factor[32 * k + 8 * g + 4 * e];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[4 * e + r] = u[2 * k + e][r], z[4 * e + r] = f[r] * u[2 * k + e][r];
      }
      split<kUParts>(y, up[k]), split<kSParts>(z, sp[k]);
    }
    const float decay = ch.decay;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      S[j] = S[j] * decay;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const v8bf f = load8(kt + (size_t)place(j, col) * C + 32 * k + 8 * g);
#pragma unroll
        for (int p = kSParts - 1; p >= 0; --p) S[j] = mfma(f, sp[k][p], S[j]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int token = place(t, col);
      o[t] = o[t] * ch.q_factor[token];
#pragma unroll
      for (int k = 0; k <= t / 2; ++k)
#pragma unroll
        for (int p = 0; p < kPParts; ++p) {
          const v8bf f = load8(&ch.p[p][token][32 * k + 8 * g]);
#pragma unroll
          for (int l = 0; l < kUParts && l + p < 2; ++l) o[t] = mfma(up[k][l], f, o[t]);
        }
      if (token < m)
        *reinterpret_cast<uint2*>(a.out + ((row0 + token) * a.Hv + h) * dv + col0 + 4 * g) =
            make_uint2(bf16x2(o[t][0], o[t][1]), bf16x2(o[t][2], o[t][3]));
    }
  }
  if (write >= 0 && write < a.s.slots)
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        a.state[write * a.s.slot_stride + at + (size_t)place(j, 4 * g + r) * dv] = S[j][r];
}

template <int DK>
hipError_t launch(DeltaArgs a, int dv, hipStream_t stream) {
  a.by_heads = divisor(a.Hv), a.by_group = divisor(a.Hv / a.Hk);
  const int chunks = a.s.total / C + a.s.batch;
  delta_prepare<DK><<<(unsigned)(chunks * a.Hv), 256, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  delta_chunks<DK><<<(unsigned)(a.s.batch * a.Hv * (dv / 64)), 256, 0, stream>>>(a, dv);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_chunks(const DeltaArgs& a, int dk, int dv, hipStream_t stream) {
  return dk == 128 ? launch<128>(a, dv, stream) : launch<64>(a, dv, stream);
}

DeltaPlan delta_plan(int total, int batch, int max_q, int write_cols, int Hk, int Hv, int dk, int dv) {
  DeltaPlan p = {};
  p.chunks = max_q > 16 && !write_cols && total > 0;
  if (p.chunks) {
    const size_t chunks = total / C + batch;
    p.kt = chunks * Hv * sizeof(ChunkHead);
    p.workspace = p.kt + chunks * Hk * dk * C * 2;
  }
  return p;
}

}  // namespace dec
