// The short causal convolution over a linear-attention layer's q, k and v channels, with SiLU and a state
// of the last width - 1 inputs of each sequence, for gfx950. 2 W + 5 operations an element against the 4 bytes
// that it is read and written with: HBM bounds it. 4500 tokens of 10240 channels: 41 us, 4.5 TB/s.
//
// A lane has 8 channels (one 16-byte load a token) and kRun consecutive tokens of a sequence, the window in
// registers. The lanes with a sequence's first tokens read its state and write the new one, which are the
// same memory where a sequence goes on in place: reading comes first in each lane, and no other lane touches
// these channels of it.
#include "decode_ops.h"
#include "dec_internal.h"

namespace dec {
namespace {

constexpr int kRun = 16;    // tokens of a lane

__device__ __forceinline__ void unpack(uint4 x, float y[8]) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) y[2 * i] = bf16_lo(u[i]), y[2 * i + 1] = bf16_hi(u[i]);
}

template <int W>
__global__ __launch_bounds__(256) void conv_rows(ConvArgs a, int runs, Divisor by_blocks, Divisor by_runs) {
  const int br = by_blocks((int)blockIdx.x);
  const int c = ((int)blockIdx.x - br * by_blocks.d) * 256 + (int)threadIdx.x;
  if (c >= a.C / 8) return;
  const int b = by_runs(br);
  int first, n;
  rows_of(a.s, b, first, n);
  float w[8][W], bias[8] = {};
#pragma unroll
  for (int i = 0; i < W; ++i) {         // 8 channels' weights, W of a channel side by side
    float y[8];
    unpack(*reinterpret_cast<const uint4*>(a.w + (size_t)c * 8 * W + 8 * i), y);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[(8 * i + j) / W][(8 * i + j) % W] = y[j];
  }
  if (a.bias) unpack(*reinterpret_cast<const uint4*>(a.bias + 8 * c), bias);
  const uint16_t* x = a.x + (size_t)first * a.x_ts + 8 * c;
  uint16_t* out = a.out + (size_t)first * a.C + 8 * c;
  const auto row = [&](int t) { return *reinterpret_cast<const uint4*>(x + (size_t)t * a.x_ts); };
  // (a sequence of more tokens than max_q takes further rounds)
  for (int t0 = (br - b * runs) * kRun; t0 == 0 || t0 < n; t0 += runs * kRun) {
    uint4 past[W - 1];
    if (t0) {
#pragma unroll
      for (int i = 0; i < W - 1; ++i) past[i] = row(t0 - (W - 1) + i);
    } else {
      const int r = a.s.read[b];
      const uint32_t fill = r < 0 ? 0u : 0x7FC07FC0u;
#pragma unroll
      for (int i = 0; i < W - 1; ++i)
        past[i] = r >= 0 && r < a.s.slots
                      ? *reinterpret_cast<const uint4*>(a.state + r * a.s.slot_stride + (size_t)i * a.C + 8 * c)
                      : make_uint4(fill, fill, fill, fill);
      // new states: the inputs up to `upto` tokens of this call
      const auto keep = [&](int slot, int upto) {
        if (slot < 0 || slot >= a.s.slots) return;
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
          const int t = upto - (W - 1) + i;
          uint4 y = past[W - 2];
          if (t >= 0) {
            y = row(t);
          } else {
#pragma unroll
            for (int p = 0; p < W - 1; ++p)
              if (t + W - 1 == p) y = past[p];
          }
          *reinterpret_cast<uint4*>(a.state + slot * a.s.slot_stride + (size_t)i * a.C + 8 * c) = y;
        }
      };
      const int* slots = a.s.write + b * a.s.write_stride;
      if (a.s.write_cols)
        for (int i = 0; i < min(n, a.s.write_cols); ++i) keep(slots[i], i + 1);
      else
        keep(slots[0], n);
    }
    float win[W][8];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) unpack(past[i], win[i]);
    const int m = min(n - t0, kRun);
    for (int t = 0; t < m; ++t) {
      unpack(row(t0 + t), win[W - 1]);
      float z[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        z[j] = bias[j];
#pragma unroll
        for (int i = 0; i < W; ++i) z[j] = fmaf(w[j][i], win[i][j], z[j]);
        if (a.silu) z[j] = z[j] / (1.0f + __expf(-z[j]));
      }
      *reinterpret_cast<uint4*>(out + (size_t)(t0 + t) * a.C) =
          make_uint4(bf16x2(z[0], z[1]), bf16x2(z[2], z[3]), bf16x2(z[4], z[5]), bf16x2(z[6], z[7]));
#pragma unroll
      for (int i = 0; i < W - 1; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) win[i][j] = win[i + 1][j];
    }
  }
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, int width, hipStream_t stream) {
  const int blocks = ceil_div(a.C / 8, 256);
  const long most = max(kMaxGrid / blocks / a.s.batch, 1L);
  const int runs = (int)min((long)max(ceil_div(min(a.s.max_q, a.s.total), kRun), 1), most);
  const unsigned grid = (unsigned)(blocks * a.s.batch * runs);
  const Divisor by_blocks = divisor(blocks), by_runs = divisor(runs);
  if (width == 2) conv_rows<2><<<grid, 256, 0, stream>>>(a, runs, by_blocks, by_runs);
  else if (width == 3) conv_rows<3><<<grid, 256, 0, stream>>>(a, runs, by_blocks, by_runs);
  else conv_rows<4><<<grid, 256, 0, stream>>>(a, runs, by_blocks, by_runs);
  return hipGetLastError();
}

}  // namespace dec
