// The gated delta rule in chunks of 64 tokens, for gfx950: the form for prompts.
//
// With G the running sum of g in a chunk, S the state before it, and k, q of unit length, the tokens' u and
// outputs are (rows are tokens)
//   (1 + A) U = diag(beta) (V - diag(e^G) K S),   A_ij = beta_i e^(G_i - G_j) k_i . k_j for j < i
//   O = scale (diag(e^G) Q S + P U),              P_ij = e^(G_i - G_j) q_i . k_j for j <= i
//   S <- e^(G_63) S + K^T diag(e^(G_63 - G)) U
// A and P do not depend on the state: delta_prepare makes T = (1 + A)^-1 diag(beta) and P of every chunk and
// head at once, and delta_chunks goes through a sequence's chunks with the state in registers.
//
// Operands are fp16. A row of K or Q is scaled by a power of two and then exact; what comes from sums in fp32 is
// scaled likewise (T and P by 2^12, columns of S, X = V - diag(e^G) K S and U by their largest element) and
// split into two parts that add up to it, the second the rounding of what the first leaves: 22 bits, and
// products of two such as three instructions. Two parts of bf16 hold 16 bits, and three of them took 182
// instructions a chunk in place of 132. A state is as far from the definition as a plain evaluation in fp32.
// T and P are at most 1 and held to 2^-37. So an output has what its own chunk adds to within 2^-37 of the values
// there, which a query or a key that is shorter than sqrt(eps) / 2^28 makes smaller than that.
//
// A wave has 16 columns of a state, which do not meet others, so that its products need no other wave. As a
// matrix instruction's result a column is a lane and 4 rows of 16 lie in a lane's registers; as its operand a
// column is a lane and 8 of the 32 terms lie in them. The sums run over whatever order of terms both
// operands have, so with rows 8 g + 4 e + r of 32 in tile e, lane group g and register r (place(), below),
// two result tiles are one operand as they are: S, X and U go from product to product without leaving their
// lanes. The other operands come from memory in the order in which lanes want them.
#include "decode_ops.h"
#include "dec_chunks.h"
#include "dec_delta.h"
#include "dec_internal.h"

namespace dec {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

constexpr int C = kChunk;
constexpr int kPad = 68;                // floats of a row of a chunk's matrices in LDS
constexpr int kFrag = 1024;             // bytes of an operand: 64 lanes of 16
constexpr int kLower = 6;               // operands of T or P: row tiles 0, 1 with terms 0..31, tiles 2, 3 with all
constexpr float kUnit = 4096.0f;        // what T and P are scaled by

// A chunk and head's part of the workspace.
struct ChunkHead {
  v8h t[2][kLower][64];
  float k_factor[C], u_factor[C];       // e^G / |k|, e^(G_63 - G) / |k|, for the scaled k
  float decay, pad[C - 1];              // e^(G_63)
  float q_factor[C];                    // e^G / |q|, for the scaled q
  v8h p[2][kLower][64];
};
constexpr int kHeadStage = 13 * kFrag;  // of it, what delta_chunks takes through LDS
// A chunk and key head's: K as rows and as columns of the products (which go through LDS), and Q.
template <int DK>
struct ChunkKeys {
  v8h k[4][DK / 32][64], kt[DK / 16][2][64], q[4][DK / 32][64];
};

// Token (or key channel) of row m of a tile: the order that makes two result tiles an operand.
__device__ __forceinline__ int place(int tile, int m) {
  return 32 * (tile >> 1) + 8 * (m >> 2) + 4 * (tile & 1) + (m & 3);
}
// Operand of row tile t and terms 32 k .. 32 k + 31 among the kLower.
__device__ __forceinline__ constexpr int lower(int t, int k) { return t < 2 ? t : 2 * t - 2 + k; }

__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ v2h half2(float a, float b) { return __builtin_convertvector(v2f{a, b}, v2h); }

// x scale as two parts that add up to it, 8 values, in two operations a value: fused multiply-adds that round
// to fp16 (scale is a power of two, so that what the first part leaves is exact).
__device__ __forceinline__ void split(const float x[8], float scale, v8h& hi, v8h& lo) {
  v4i a, b;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const v2h part = {(_Float16)__builtin_fmaf(x[i], scale, 0.0f), (_Float16)__builtin_fmaf(x[i + 1], scale, 0.0f)};
    int bits = __builtin_bit_cast(int, part);
    asm("" : "+v"(bits));               // (both halves are read from here)
    a[i / 2] = bits;
    const v2h first = __builtin_bit_cast(v2h, bits);
    b[i / 2] = __builtin_bit_cast(int, v2h{(_Float16)__builtin_fmaf(x[i], scale, -(float)first[0]),
                                           (_Float16)__builtin_fmaf(x[i + 1], scale, -(float)first[1])});
  }
  hi = __builtin_bit_cast(v8h, a), lo = __builtin_bit_cast(v8h, b);
}

// The power of two that brings a magnitude (its bits) to 2^13 .. 2^14, and one over it. What is below 2^-113
// counts as that; what is not finite stays so.
__device__ __forceinline__ float scale_to(uint32_t top) { return __uint_as_float((267u - max(top >> 23, 14u)) << 23); }
__device__ __forceinline__ float scale_back(uint32_t top) { return __uint_as_float((max(top >> 23, 14u) - 13u) << 23); }

__device__ __forceinline__ float larger(float top, float x) { return fmaxf(top, fabsf(x)); }
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Over the four lanes that have the same column (or row).
__device__ __forceinline__ uint32_t max_groups(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}
__device__ __forceinline__ float sum_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t y = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ v4i load8(const uint16_t* p) { return *reinterpret_cast<const v4i*>(p); }
// Element i of 8 bf16.
__device__ __forceinline__ float element(v4i x, int i) { return i & 1 ? bf16_hi((uint32_t)x[i / 2]) : bf16_lo((uint32_t)x[i / 2]); }

// Keys and queries of a chunk slot and key head, behind the heads' parts.
template <int DK>
__device__ __forceinline__ ChunkKeys<DK>& delta_keys(const DeltaArgs& a, int c, int hk) {
  return ((ChunkKeys<DK>*)((char*)a.workspace + a.keys))[(size_t)c * a.Hk + hk];
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ double wave_sums(double x) {
#define STEP(ctrl, rows)                                                                                      \
  {                                                                                                           \
    const uint64_t u = (uint64_t)__double_as_longlong(x);                                                     \
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, ctrl, rows, 0xF, false);    \
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), ctrl, rows, 0xF, false); \
    x += __longlong_as_double((long long)((uint64_t)hi << 32 | lo));                                          \
  }
  STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF)     // row_shr:1, 2, 4, 8
  STEP(0x142, 0xA) STEP(0x143, 0xC)                                       // row_bcast:15 and 31
#undef STEP
  return x;
}

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

template <int DK>
struct PrepareShared {
  float a[C][kPad];
  union {
    float t[C][kPad];
    v8h k[4][DK / 32][64];              // K until its products are formed
  };
  float g_hi[C], g_lo[C], beta[C], rk[C], rq[C];           // G in units of ln 2
};

// One workgroup makes one chunk's matrices for one value head; wave w has rows 16 w .. 16 w + 15.
template <int DK>
__global__ __launch_bounds__(256, 4) void delta_prepare(DeltaArgs a) {
  __shared__ __attribute__((aligned(16))) PrepareShared<DK> s;
  const int c = a.by_heads((int)blockIdx.x), h = (int)blockIdx.x - c * a.Hv;
  const int hk = a.by_group(h);
  size_t row0;
  int m;
  if (!rows_of_chunk(a.s, c, row0, m)) return;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;

  constexpr int kSteps = DK / 32;
  uint16_t gate_a = 0, gate_b = 0;
  if (w == 0) {
    const size_t row = row0 + min(lane, m - 1);
    gate_a = a.a[row * a.a_ts + h], gate_b = a.b[row * a.b_ts + h];
  }
  v4i raw_k[kSteps], raw_q[kSteps];
  {
    const size_t row = row0 + min(16 * w + col, m - 1);
    const uint16_t* k = a.k + row * a.k_ts + hk * a.k_hs + 8 * g;
    const uint16_t* q = a.q + row * a.q_ts + hk * a.q_hs + 8 * g;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) raw_k[i] = load8(k + 32 * i);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) raw_q[i] = load8(q + 32 * i);
  }
  if (w == 0) {
    // (decays below e^-200 are 0 either way; held to that, the sums stay finite)
    const float x = log_decay(bf16_f32(gate_a), decay_rate(a.a_log[h]), a.dt_bias[h]);
    const double sum = wave_sums(lane < m ? (double)(x < -200.0f ? -200.0f : x) * 1.4426950408889634 : 0.0);
    // two floats: differences of nearby sums keep the bits of what lies between them
    s.g_hi[lane] = (float)sum, s.g_lo[lane] = (float)(sum - (double)(float)sum);
    s.beta[lane] = lane < m ? sigmoid(bf16_f32(gate_b)) : 0.0f;
  }
  // rows scaled to fp16, one over their lengths
  const auto scaled = [&](const v4i x[kSteps], v8h y[kSteps]) {
    typedef uint16_t v2u __attribute__((ext_vector_type(2)));
    v2u most = {};
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2u, x[i][j] & 0x7FFF7FFF));
    const float scale = scale_to(max_groups((uint32_t)max(most[0], most[1]) << 16));
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float z = element(x[i], j) * scale, z1 = element(x[i], j + 1) * scale;
        const v2h both = half2(z, z1);
        y[i][j] = both[0], y[i][j + 1] = both[1], squares = fmaf(z1, z1, fmaf(z, z, squares));
      }
    return over_length(1.0f, sum_groups(squares), a.eps, scale);
  };
  v8h kf[kSteps], qf[kSteps];
  const float rk = scaled(raw_k, kf);
  __builtin_amdgcn_sched_barrier(0);    // (one after the other: both at once spill)
  const float rq = scaled(raw_q, qf);
  if (g == 0) s.rk[16 * w + col] = rk, s.rq[16 * w + col] = rq;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) s.k[w][i][lane] = kf[i];
  __syncthreads();
  v4f p[4];
  {
    const v4f rki = *(const v4f*)&s.rk[16 * w + 4 * g], rqi = *(const v4f*)&s.rq[16 * w + 4 * g];
    const v4f hi = *(const v4f*)&s.g_hi[16 * w + 4 * g], lo = *(const v4f*)&s.g_lo[16 * w + 4 * g];
    const v4f beta = *(const v4f*)&s.beta[16 * w + 4 * g];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t > (w | 1)) break;
      v4f ak = {}, aq = {};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const v8h x = s.k[t][i][lane];
        ak = mfma(kf[i], x, ak), aq = mfma(qf[i], x, aq);
      }
      const int j = 16 * t + col;
      const float hj = s.g_hi[j], lj = s.g_lo[j], rkj = s.rk[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * w + 4 * g + r;
        const float d = j <= i ? exp2_raw((hi[r] - hj) + (lo[r] - lj)) * rkj : 0.0f;
        s.a[i][j] = j < i ? beta[r] * d * rki[r] * ak[r] : 0.0f;
        p[t][r] = j <= i ? d * rqi[r] * aq[r] : 0.0f;
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
      asm volatile("" : "+v"(t[i]) : : "memory");     // (all rows read at once would spill)
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
#pragma unroll
  for (int t = 0; t < 4; ++t)
    if (t <= (w | 1))
#pragma unroll
      for (int r = 0; r < 4; ++r) s.a[16 * w + 4 * g + r][16 * t + col] = p[t][r];
  __syncthreads();
  ChunkHead& out = ((ChunkHead*)a.workspace)[(size_t)c * a.Hv + h];
#pragma unroll
  for (int x = tid; x < 2 * kLower * 64; x += 256) {
    const bool is_p = x >= kLower * 64;
    const int f = (is_p ? x - kLower * 64 : x) >> 6;       // operand, and its row tile and terms
    const int t = f < 2 ? f : 2 + (f - 2) / 2, k = f < 2 ? 0 : (f - 2) & 1;
    const int i = place(t, col), j = 32 * k + 8 * g;
    float y[8];
#pragma unroll
    for (int l = 0; l < 8; ++l) y[l] = is_p ? s.a[i][j + l] : s.t[i][j + l] * s.beta[j + l];
    v8h hi, lo;
    split(y, kUnit, hi, lo);
    v8h(*to)[kLower][64] = is_p ? out.p : out.t;
    to[0][f][lane] = hi, to[1][f][lane] = lo;
  }
  if (w == 0) {
    const float hi = s.g_hi[lane], lo = s.g_lo[lane], last = s.g_hi[C - 1], rest = s.g_lo[C - 1];
    const float in = exp2_raw(hi + lo), there = lane < m ? 1.0f : 0.0f;
    out.k_factor[lane] = there * (in * s.rk[lane]);
    out.q_factor[lane] = in * s.rq[lane];
    out.u_factor[lane] = there * (exp2_raw((last - hi) + (rest - lo)) * s.rk[lane]);
    if (lane == 0) out.decay = exp2_raw(last + rest);
  }
  if (hk * (a.Hv / a.Hk) == h) {        // K and Q once for the heads that share them
    ChunkKeys<DK>& keys = delta_keys<DK>(a, c, hk);
    const int token = 16 * w + col, tile = 2 * (token >> 5) + ((token >> 2) & 1);
    const int row = 4 * ((token >> 3) & 3) + (token & 3);
    __syncthreads();
    _Float16(*kt)[C + 8] = (_Float16(*)[C + 8]) s.a;       // [DK][C], over a and t
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const v8h x = kf[step];
      keys.k[tile][step][16 * g + row] = x;
      keys.q[tile][step][16 * g + row] = qf[step];
#pragma unroll
      for (int l = 0; l < 8; ++l) kt[32 * step + 8 * g + l][token] = x[l];
    }
    __syncthreads();
#pragma unroll
    for (int x = tid; x < DK / 8 * 64; x += 256) {
      const int j = x >> 7, k = (x >> 6) & 1;
      keys.kt[j][k][lane] = *(const v8h*)&kt[place(j, col)][32 * k + 8 * g];
    }
  }
}

// The last word of a buffer descriptor: plain bytes, loads past its end give zero.
constexpr int kBufferWord3 = 0x00020000;

// 64 lanes of 16 bytes, offset bytes behind a buffer's beginning.
template <typename Buffer>
__device__ __forceinline__ v8h load_frag(Buffer p, int lane16, int offset) {
  return __builtin_bit_cast(v8h, __builtin_amdgcn_raw_buffer_load_b128(p, lane16, offset, 0));
}

__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// LDS reads above this are not moved below it, nor those below above.
__device__ __forceinline__ void hold_reads() { __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x8 | 0x10 | 0x200 | 0x400); }

// N times a matrix instruction and three vector instructions.
template <int N>
__device__ __forceinline__ void mix_products() {
  if constexpr (N > 0) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);
    mix_products<N - 1>();
  }
}

// Waits for all loads but the last N.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));   // vmcnt(N)
  asm volatile("" ::: "memory");
}

// What the waves of a workgroup of delta_chunks share.
template <int DK, int NW>
struct ChunkShared {
  struct Stage {
    union {
      struct {
        v8h t[2][kLower][64];
        float k_factor[C], u_factor[C], decay, pad[C - 1], unused[C];
      };
      char head[kHeadStage];
    };
    v8h k[4][DK / 32][64], kt[DK / 16][2][64];
  } stage[3];
  struct {
    v8h s[2][DK / 32][64];              // parts of the state before the chunk
    v4f u[4][64];                       // U of the chunk, and before that its values
    float s_back[16], x_back[16], u_back[16];      // one over the columns' scales
  } wave[NW];
};

// A workgroup has 16 NW columns of a sequence and head's state. Waves 0 .. NW - 1 have 16 of them each and go
// through the chunks; wave NW + i makes the outputs of wave i's columns, a chunk behind, and moves the next
// chunk's operands to LDS.
template <int DK, int NW>
__global__ __launch_bounds__(128 * NW) __attribute__((amdgpu_waves_per_eu(NW / 2, NW / 2)))
void delta_chunks(DeltaArgs a, int dv, int parts, int sequences) {
  constexpr int kSteps = DK / 32, kTiles = DK / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  ChunkShared<DK, NW>& sh = *(ChunkShared<DK, NW>*)lds;
  // a head's parts on one of the 8 dies, which have an L2 each
  const int part = (int)(blockIdx.x >> 3) % parts, bh = (int)(blockIdx.x >> 3) / parts * 8 + (int)(blockIdx.x & 7);
  if (bh >= sequences) return;
  const int b = a.by_heads(bh), h = bh - b * a.Hv, hk = a.by_group(h);
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool outputs = wave >= NW;
  const int mine = outputs ? wave - NW : wave;
  const int col0 = (part * NW + mine) * 16;
  auto& ex = sh.wave[mine];
  int first, n;
  rows_of(a.s, b, first, n);
  const int chunks = ceil_div(n, kChunk), c0 = first_chunk(a.s, b);
  const auto head_of = [&](int c) -> const ChunkHead& { return ((const ChunkHead*)a.workspace)[(size_t)(c0 + c) * a.Hv + h]; };

  if (outputs) {
    // operands of chunk c to stage c % 3, this wave's share of them
    const int lane16 = lane * 16;
    constexpr int kHead = kHeadStage / kFrag, kKeys = 4 * kSteps + 2 * kTiles;
    const auto move = [&](int c) {
      const auto head = __builtin_amdgcn_make_buffer_rsrc((char*)&head_of(c) + mine * kFrag, 0, kHeadStage - mine * kFrag, kBufferWord3);
      const auto keys = __builtin_amdgcn_make_buffer_rsrc((char*)&delta_keys<DK>(a, c0 + c, hk) + mine * kFrag, 0, kKeys * kFrag, kBufferWord3);
      char* to = sh.stage[c % 3].head + mine * kFrag;
      char* to_keys = (char*)sh.stage[c % 3].k + mine * kFrag;
#pragma unroll
      for (int x = 0; x < kKeys; x += NW)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(keys, (lds_ptr)(to_keys + x * kFrag), 16, lane16, x * kFrag, 0, 0);
#pragma unroll
      for (int x = 0; x < kHead; x += NW)
        if (x + NW <= kHead || x + mine < kHead)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(head, (lds_ptr)(to + x * kFrag), 16, lane16, x * kFrag, 0, 0);
    };
    // values of chunk c, rows as results have them; rows past the sequence read as zero
    uint16_t raw[16];
    v4f v[4];
    const int v_row = (int)a.v_ts * 2, v_at = 8 * g * v_row + 2 * col;
    const auto load_v = [&](int c) {
      const auto from = __builtin_amdgcn_make_buffer_rsrc((void*)(a.v + ((size_t)first + c * C) * a.v_ts + h * a.v_hs + col0), 0,
                                                          (min(n - c * C, C) - 1) * v_row + 32, kBufferWord3);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        raw[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(from, v_at + place(i >> 2, i & 3) * v_row, 0, 0);
    };
    const auto take_v = [&] {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i >> 2][i & 3] = bf16_f32(raw[i]);
    };
    const auto give_v = [&] {
#pragma unroll
      for (int t = 0; t < 4; ++t) ex.u[t][lane] = v[t];
    };
    v8h q[4][kSteps], p[2][kLower], sp[2][kSteps];
    v4f u[4], s_back;
    float q_factor[4], o_factor[4], x_back;
    const auto load = [&](int c) {
      const auto head = __builtin_amdgcn_make_buffer_rsrc((void*)&head_of(c), 0, (int)sizeof(ChunkHead), kBufferWord3);
      const auto keys = __builtin_amdgcn_make_buffer_rsrc((void*)delta_keys<DK>(a, c0 + c, hk).q, 0, (int)sizeof(ChunkKeys<DK>::q), kBufferWord3);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        q_factor[t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            head, 4 * place(t, col), offsetof(ChunkHead, q_factor), 0));
#pragma unroll
        for (int i = 0; i < kSteps; ++i) q[t][i] = load_frag(keys, lane16, (t * kSteps + i) * kFrag);
      }
#pragma unroll
      for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int f = 0; f < kLower; ++f)
          p[l][f] = load_frag(head, lane16, (int)offsetof(ChunkHead, p) + (l * kLower + f) * kFrag);
    };
    if (chunks > 0) load_v(0), move(0);
    if (chunks > 1) move(1);
    if (chunks > 0) take_v(), give_v();
    if (chunks > 1) load_v(1);
    wait_loads<0>();
    lds_barrier();                      // stage 0 and its values are there
    for (int c = 0; c <= chunks; ++c) {
      lds_barrier();                    // A: all have taken what chunk c - 1 left
      uint32_t top = 0;
      if (c > 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = max(top, magnitude(u[t][r]));
        top = max_groups(top);
      }
      const bool mine_to_write = c > 0 && !__any(top >= 0x7F800000u);    // (else the other wave writes them)
      v4f o[4] = {}, x[4] = {};
      if (mine_to_write) {
        // outputs of chunk c - 1: rows are columns of the state, columns tokens
        const float up = scale_to(top);
        if (g == 0) ex.u_back[col] = scale_back(top) * x_back * (1.0f / kUnit);
        v8h uh[2], ul[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = u[2 * k + i / 4][i & 3];
          split(y, up, uh[k], ul[k]);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int l = 1; l >= 0; --l)
#pragma unroll
            for (int t = 0; t < 4; ++t) o[t] = mfma(sp[l][i], q[t][i], o[t]);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int l = 0; l < 3; ++l)
#pragma unroll
            for (int t = 2 * k; t < 4; ++t)
              x[t] = mfma(l == 0 ? ul[k] : uh[k], p[l == 1][lower(t, k)], x[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) o_factor[t] = a.scale * q_factor[t];
      }
      wait_loads<0>();                  // stage c + 1 is there
      if (c + 1 < chunks) take_v();
      if (c < chunks) load(c);
      if (c + 2 < chunks) load_v(c + 2);
      if (mine_to_write) {
        const v4f u_back = *(const v4f*)&ex.u_back[4 * g] * a.scale;
        const int m = min(n - (c - 1) * C, C);
        uint16_t* out = a.out + (((size_t)first + (c - 1) * C) * a.Hv + h) * dv + col0 + 4 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int token = place(t, col);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][r] = fmaf(o[t][r], s_back[r] * o_factor[t], x[t][r] * u_back[r]);
          if (token < m)
            *reinterpret_cast<uint2*>(out + (size_t)token * a.Hv * dv) =
                make_uint2(bf16x2(o[t][0], o[t][1]), bf16x2(o[t][2], o[t][3]));
        }
      }
      if (c == chunks) break;
      lds_barrier();                    // B: wave `mine` has left what the outputs of chunk c take
      x_back = ex.x_back[col];
      s_back = *(const v4f*)&ex.s_back[4 * g];
#pragma unroll
      for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int i = 0; i < kSteps; ++i) sp[l][i] = ex.s[l][i][lane];
#pragma unroll
      for (int t = 0; t < 4; ++t) u[t] = ex.u[t][lane];
      if (c + 1 < chunks) give_v();
      if (c + 2 < chunks) move(c + 2);  // (to where chunk c - 1 was, which all are through with)
    }
    return;
  }

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
  // What chunk c adds to the state, K^T U, is formed with the products that chunk c + 1 takes of it, tile
  // pair after tile pair: the vector instructions on one pair under the matrix instructions on the next.
  v8h uh[2], ul[2];                     // U of the chunk before, decayed to its end
  float u_back = 0.0f, decay = 0.0f, u_most = 0.0f, s_top = 0.0f;
  bool adds = false;
  const auto added = [&](const v8h kt[2][2], v4f y[2]) {
#pragma unroll
    for (int e = 0; e < 2; ++e) y[e] = v4f{};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int l = 1; l >= 0; --l)
#pragma unroll
        for (int e = 0; e < 2; ++e) y[e] = mfma(kt[e][k], l ? ul[k] : uh[k], y[e]);
  };
  const auto add = [&](int i, const v4f y[2]) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[2 * i + e][r] = fmaf(S[2 * i + e][r], decay, y[e][r] * u_back);
  };
  lds_barrier();                        // (stage 0 is there)
  for (int c = 0, place_of = 0, last = 2; c < chunks; ++c) {
    const auto& st = sh.stage[place_of];
    const auto& before = sh.stage[last];
    last = place_of, place_of = place_of == 2 ? 0 : place_of + 1;
    const int m = min(n - c * C, C);
    v8h kf[2][4], kt[3][2][2], tf[2][kLower];
    const auto read_k = [&](int i) {
#pragma unroll
      for (int t = 0; t < 4; ++t) kf[i & 1][t] = st.k[t][i][lane];
    };
    const auto read_kt = [&](int i) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) kt[i % 3][e][k] = before.kt[2 * i + e][k][lane];
    };
    read_kt(0), read_k(0), read_kt(1);
    hold_reads();
    v4f y[2][2];
    if (adds) added(kt[0], y[0]);
    lds_barrier();                      // A
    v4f v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = ex.u[t][lane];
    // The scale of the state's columns: by their largest element, or where the state is still to be
    // formed by a bound of it, decay max |S| + 64 max |u| (keys are no longer than 1).
    if (!adds) {
      s_top = 0.0f;
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_top = larger(s_top, S[j][r]);
      s_top = __uint_as_float(max_groups(__float_as_uint(s_top)));
    }
    const uint32_t bound = __float_as_uint(adds ? fmaf(decay, s_top, 64.0f * u_most) : s_top);
    const float s_to = scale_to(bound), s_back = scale_back(bound);
    if (g == 0) ex.s_back[col] = s_back;
    s_top = 0.0f;
    v4f x[4] = {};
    v8h sh_[2], sl[2];
    const auto parts_of = [&](int i) {
      float y[8];
#pragma unroll
      for (int l = 0; l < 8; ++l) y[l] = S[2 * i + l / 4][l & 3], s_top = larger(s_top, y[l]);
      split(y, s_to, sh_[i & 1], sl[i & 1]);
      ex.s[0][i][lane] = sh_[i & 1], ex.s[1][i][lane] = sl[i & 1];
    };
    const auto products = [&](int i) {
#pragma unroll
      for (int l = 1; l >= 0; --l)
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = mfma(kf[i & 1][t], l ? sl[i & 1] : sh_[i & 1], x[t]);
    };
    const auto read_t = [&](int l) {
#pragma unroll
      for (int f = 0; f < kLower; ++f) tf[l][f] = st.t[l][f][lane];
    };
    // Operands are read a step before their products: alone on its SIMD, a wave waits for every read. The
    // products that a step issues do not depend on its vector instructions, which go between them.
    if (adds) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (i + 2 < kSteps) read_kt(i + 2);
        if (i == kSteps - 2) read_t(0);
        if (i == kSteps - 1) read_t(1);
        hold_reads();
        if (i > 0) products(i - 1);
        if (i + 1 < kSteps) added(kt[(i + 1) % 3], y[(i + 1) & 1]);
        add(i, y[i & 1]);
        parts_of(i);
        mix_products<16>();
        if (i + 1 < kSteps) read_k(i + 1);
      }
      products(kSteps - 1);
    } else {
      read_t(0), read_t(1);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (i + 1 < kSteps) read_k(i + 1);
        parts_of(i);
        products(i);
      }
    }
    s_top = __uint_as_float(max_groups(__float_as_uint(s_top)));
    float x_top = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const v4f f = *(const v4f*)&st.k_factor[place(t, 4 * g)];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[t][r] = fmaf(-(f[r] * s_back), x[t][r], v[t][r]);
        x_top = larger(x_top, x[t][r]);
      }
    }
    const uint32_t x_most = max_groups(__float_as_uint(x_top));
    const float x_to = scale_to(x_most), x_back = scale_back(x_most) * (1.0f / kUnit);
    if (g == 0) ex.x_back[col] = x_back;
    v8h xh[2], xl[2];
    v4f u[4] = {};                      // U, in X's scale
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
#pragma unroll
      for (int l = 0; l < 8; ++l) y[l] = x[2 * k + l / 4][l & 3];
      split(y, x_to, xh[k], xl[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int l = 0; l < 3; ++l)       // small products first
#pragma unroll
        for (int t = 2 * k; t < 4; ++t)
          u[t] = mfma(tf[l == 1][lower(t, k)], l == 0 ? xl[k] : xh[k], u[t]);
    uint32_t top = 0;
    float f_top = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      ex.u[t][lane] = u[t];
      const v4f f = *(const v4f*)&st.u_factor[place(t, 4 * g)];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        top = max(top, magnitude(u[t][r]));
        u[t][r] *= f[r], f_top = larger(f_top, u[t][r]);
      }
    }
    top = max_groups(top);
    lds_barrier();                      // B
    if (__any(top >= 0x7F800000u)) {
      adds = false;                     // (the state is the one before this chunk by now)
      // Something is not finite: token after token, so that no token sees a later one through a product
      // with zero.
      const float rate = decay_rate(a.a_log[h]), dt = a.dt_bias[h];
      for (int t = 0; t < m; ++t) {
        const size_t row = (size_t)first + c * C + t;
        const float alpha = expf(log_decay(bf16_f32(a.a[row * a.a_ts + h]), rate, dt));
        const float beta = sigmoid(bf16_f32(a.b[row * a.b_ts + h]));
        const float vt = bf16_f32(a.v[row * a.v_ts + h * a.v_hs + col0 + col]);
        float kk = 0.0f, qq = 0.0f, sk = 0.0f, sq = 0.0f, kt = 0.0f, qt = 0.0f;
        v4i kf[kSteps], qf[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          kf[i] = load8(a.k + row * a.k_ts + hk * a.k_hs + 32 * i + 8 * g);
          qf[i] = load8(a.q + row * a.q_ts + hk * a.q_hs + 32 * i + 8 * g);
#pragma unroll
          for (int l = 0; l < 8; ++l) kt = larger(kt, element(kf[i], l)), qt = larger(qt, element(qf[i], l));
        }
        const float pk = unit_power(__uint_as_float(max_groups(__float_as_uint(kt))));
        const float pq = unit_power(__uint_as_float(max_groups(__float_as_uint(qt))));
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int l = 0; l < 8; ++l) {
            const float kx = element(kf[i], l) * pk, qx = element(qf[i], l) * pq;
            kk = fmaf(kx, kx, kk), qq = fmaf(qx, qx, qq), sk = fmaf(S[2 * i + l / 4][l & 3], kx, sk);
          }
        kk = sum_groups(kk), qq = sum_groups(qq), sk = sum_groups(sk);
        const float rk = over_length(1.0f, kk, a.eps, pk), rq = over_length(a.scale, qq, a.eps, pq);
        const float ut = beta * (vt - alpha * rk * sk) * rk;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int l = 0; l < 8; ++l) {
            const float y = fmaf(element(kf[i], l) * pk, ut, alpha * S[2 * i + l / 4][l & 3]);
            S[2 * i + l / 4][l & 3] = y;
            sq = fmaf(y, element(qf[i], l) * pq, sq);
          }
        sq = rq * sum_groups(sq);
        if (g == 0) a.out[(row * a.Hv + h) * dv + col0 + col] = (uint16_t)bf16x2(sq, sq);
      }
      continue;
    }
    const uint32_t f_most = max_groups(__float_as_uint(f_top));
    const float u_to = scale_to(f_most);
    u_back = scale_back(f_most) * x_back, u_most = __uint_as_float(top) * x_back, decay = st.decay;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y[8];
#pragma unroll
      for (int l = 0; l < 8; ++l) y[l] = u[2 * k + l / 4][l & 3];
      split(y, u_to, uh[k], ul[k]);
    }
    adds = true;
  }
  if (adds) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      v8h kt[2][2];
      v4f y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) kt[e][k] = sh.stage[(chunks + 2) % 3].kt[2 * i + e][k][lane];
      added(kt, y);
      add(i, y);
    }
  }
  lds_barrier();                        // (the other waves' last A)
  if (write >= 0 && write < a.s.slots)
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        a.state[write * a.s.slot_stride + at + (size_t)place(j, 4 * g + r) * dv] = S[j][r];
}

template <int DK, int NW>
hipError_t launch_chunks(const DeltaArgs& a, int dv, hipStream_t stream) {
  const int parts = dv / (16 * NW), sequences = a.s.batch * a.Hv;
  constexpr int kBytes = sizeof(ChunkShared<DK, NW>);
  static_assert(kBytes <= 160 * 1024, "LDS of a workgroup");
  if (hipError_t e = hipFuncSetAttribute((const void*)delta_chunks<DK, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, kBytes)) return e;
  delta_chunks<DK, NW><<<(unsigned)(ceil_div(sequences, 8) * 8 * parts), 128 * NW, kBytes, stream>>>(a, dv, parts, sequences);
  return hipGetLastError();
}

template <int DK>
hipError_t launch(DeltaArgs a, int dv, hipStream_t stream) {
  a.by_heads = divisor(a.Hv), a.by_group = divisor(a.Hv / a.Hk);
  const int chunks = a.s.total / C + a.s.batch;
  delta_prepare<DK><<<(unsigned)(chunks * a.Hv), 256, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  return launch_chunks<DK, 2>(a, dv, stream);
}

}  // namespace

hipError_t launch_delta_chunks(const DeltaArgs& a, int dk, int dv, hipStream_t stream) {
  return dk == 128 ? launch<128>(a, dv, stream) : launch<64>(a, dv, stream);
}

DeltaPlan delta_plan(int total, int batch, int max_q, int write_cols, int Hk, int Hv, int dk, int dv) {
  DeltaPlan p = {};
  // Token after token takes 1.6 us a token at least, in chunks 2.3 a chunk and two launches, whatever a chunk holds: 4001
  // tokens 7374 us against 188. Where they meet depends on how many workgroups there are. us, token after token and in
  // chunks, at 16, 24 and 32 tokens a sequence: 1 sequence of 48 heads 31 43 55, 17 17 17 (8 tokens: 18, 17); 8 of
  // them 44 61 78, 46 46 46; 61 of 8 heads 46 64 81, 57 57 56; 61 of 48 heads 191 267 348, 294 297 301. The rule looks at
  // the longest sequence alone, so that all go one way: 61 of one token beside one of 17 take 289, in two calls 85.
  p.chunks = max_q > 16 && !write_cols && total > 0;
  if (p.chunks) {
    const size_t chunks = total / C + batch;
    p.keys = chunks * Hv * sizeof(ChunkHead);
    p.workspace = p.keys + chunks * Hk * (dk == 128 ? sizeof(ChunkKeys<128>) : sizeof(ChunkKeys<64>));
  }
  return p;
}

}  // namespace dec
