// The gated delta rule token after token, for gfx950: the form for decoded and drafted tokens.
//
// For one value head, with the state S [dk][dv]: S <- e^g S, u = beta (v - S^T k), S <- S + k u^T, o = scale
// S^T q. The columns of S do not meet, so a wave has 32 of them: 8 lanes of 4 columns, 8 lanes of dk / 8 rows,
// the state in registers from the first token to the last. Both products of a token, S^T k and S^T q, are
// taken of the state before it and summed over the rows together, since
//   o = scale (e^g S^T q + (k . q) u).
// One token reads and writes the state once, 8 bytes an element against 7 operations: HBM bounds it. 61 sequences of 48
// heads of 128 x 128: 92 us a call, 4.2 TB/s; the squares are added, and rows of unusual length scaled, before the
// products with the state (in a loop around both, it took 106).
#include "decode_ops.h"
#include "dec_delta.h"
#include "dec_internal.h"

namespace dec {
namespace {

// Sum over the 8 lanes that have the same columns.
__device__ __forceinline__ float sum_rows(float x) {
  x += __shfl_xor(x, 8);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float max_rows(float x) {
  x = fmaxf(x, __shfl_xor(x, 8));
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

template <int R>
__device__ __forceinline__ void load_rows(const uint16_t* p, float y[R]) {
#pragma unroll
  for (int i = 0; i < R; i += 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(p + i);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) y[i + 2 * j] = bf16_lo(u[j]), y[i + 2 * j + 1] = bf16_hi(u[j]);
  }
}

template <int DK, int DV>
__global__ __launch_bounds__(256) void delta_steps(DeltaArgs a, int units) {
  constexpr int R = DK / 8, kTiles = DV / 32;
  const int unit = (int)(blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64);
  if (unit >= units) return;
  const int lane = threadIdx.x & 63, rows = (lane >> 3) * R;
  const int bh = unit / kTiles, col = (unit % kTiles) * 32 + (lane & 7) * 4;
  const int b = a.by_heads(bh), h = bh - b * a.Hv;
  const int hk = a.by_group(h);
  int first, n;
  rows_of(a.s, b, first, n);
  const size_t at = ((size_t)h * DK + rows) * DV + col;
  const int r = a.s.read[b];
  v4f S[R];
  const float fill = r < 0 ? 0.0f : __uint_as_float(0x7FC00000u);
#pragma unroll
  for (int i = 0; i < R; ++i)
    S[i] = r >= 0 && r < a.s.slots
               ? *reinterpret_cast<const v4f*>(a.state + r * a.s.slot_stride + at + (size_t)i * DV)
               : v4f{fill, fill, fill, fill};
  const int* slots = a.s.write + b * a.s.write_stride;
  const auto keep = [&](int slot) {
    if (slot < 0 || slot >= a.s.slots) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
      *reinterpret_cast<v4f*>(a.state + slot * a.s.slot_stride + at + (size_t)i * DV) = S[i];
  };
  const float rate = decay_rate(a.a_log[h]), dt = a.dt_bias[h];
  for (int t = first; t < first + n; ++t) {
    float k[R], q[R];
    load_rows<R>(a.k + (size_t)t * a.k_ts + hk * a.k_hs + rows, k);
    load_rows<R>(a.q + (size_t)t * a.q_ts + hk * a.q_hs + rows, q);
    const uint2 vv = *reinterpret_cast<const uint2*>(a.v + (size_t)t * a.v_ts + h * a.v_hs + col);
    const float v[4] = {bf16_lo(vv.x), bf16_hi(vv.x), bf16_lo(vv.y), bf16_hi(vv.y)};
    const float alpha = expf(log_decay(bf16_f32(a.a[(size_t)t * a.a_ts + h]), rate, dt));
    const float beta = sigmoid(bf16_f32(a.b[(size_t)t * a.b_ts + h]));
    float kk = 0.0f, qq = 0.0f, kq = 0.0f, sk[4] = {}, sq[4] = {}, pk = 1.0f, pq = 1.0f;
    const auto squares = [&] {
      kk = qq = 0.0f;
#pragma unroll
      for (int i = 0; i < R; ++i) kk = fmaf(k[i], k[i], kk), qq = fmaf(q[i], q[i], qq);
      kk = sum_rows(kk), qq = sum_rows(qq);
    };
    squares();
    if (!(plain_squares(kk) && plain_squares(qq))) {    // (of all lanes or none: they have the same row)
      float kt = 0.0f, qt = 0.0f;
#pragma unroll
      for (int i = 0; i < R; ++i) kt = fmaxf(kt, fabsf(k[i])), qt = fmaxf(qt, fabsf(q[i]));
      pk = unit_power(max_rows(kt)), pq = unit_power(max_rows(qt));
#pragma unroll
      for (int i = 0; i < R; ++i) k[i] *= pk, q[i] *= pq;
      squares();
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      kq = fmaf(k[i], q[i], kq);
#pragma unroll
      for (int c = 0; c < 4; ++c) sk[c] = fmaf(S[i][c], k[i], sk[c]), sq[c] = fmaf(S[i][c], q[i], sq[c]);
    }
    kq = sum_rows(kq);
#pragma unroll
    for (int c = 0; c < 4; ++c) sk[c] = sum_rows(sk[c]), sq[c] = sum_rows(sq[c]);
    const float rk = over_length(1.0f, kk, a.eps, pk), rq = over_length(a.scale, qq, a.eps, pq);
    float u[4], o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = beta * (v[c] - alpha * rk * sk[c]) * rk;    // times 1 / |k|, for the k below, not of unit length
      o[c] = rq * fmaf(kq, u[c], alpha * sq[c]);
#pragma unroll
      for (int i = 0; i < R; ++i) S[i][c] = fmaf(k[i], u[c], alpha * S[i][c]);
    }
    if (lane < 8)
      *reinterpret_cast<uint2*>(a.out + ((size_t)t * a.Hv + h) * DV + col) =
          make_uint2(bf16x2(o[0], o[1]), bf16x2(o[2], o[3]));
    if (t - first < a.s.write_cols) keep(slots[t - first]);
  }
  if (!a.s.write_cols) keep(slots[0]);
}

template <int DK, int DV>
hipError_t launch(DeltaArgs a, hipStream_t stream) {
  const int units = a.s.batch * a.Hv * (DV / 32);
  a.by_heads = divisor(a.Hv), a.by_group = divisor(a.Hv / a.Hk);
  const int waves = 4;
  delta_steps<DK, DV><<<(unsigned)ceil_div(units, waves), waves * 64, 0, stream>>>(a, units);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_steps(const DeltaArgs& a, int dk, int dv, hipStream_t stream) {
  if (dk == 128) return dv == 128 ? launch<128, 128>(a, stream) : launch<128, 64>(a, stream);
  return dv == 128 ? launch<64, 128>(a, stream) : launch<64, 64>(a, stream);
}

}  // namespace dec
