// Internals shared by the kernels of libdecode_ops.so for gfx950 (CDNA4). Not part of the C ABI
// (decode_ops.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kv4_internal.h"   // vector types, bf16 conversions, Divisor

namespace dec {

using kv4::bf16_hi;
using kv4::bf16_lo;
using kv4::bf16x2;
using kv4::bits_f32;
using kv4::ceil_div;
using kv4::Divisor;
using kv4::divisor;
using kv4::kCUs;
using kv4::v2f;
using kv4::v4f;
using kv4::v4i;
using kv4::v8bf;

__device__ __forceinline__ float bf16_f32(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }

// Workgroups of 256 threads that one launch may have: its threads are counted in 32 bits.
constexpr long kMaxGrid = (1L << 32) / 256 - 1;

// Sequences of a batch and the slots of their states.
struct Sequences {
  const int* starts;
  const int* read;
  const int* write;
  long write_stride, slots, slot_stride;
  int write_cols, total, batch, max_q;
};

// First row and number of rows of sequence b, in [0, total] whatever the starts hold.
__device__ __forceinline__ void rows_of(const Sequences& s, int b, int& first, int& n) {
  first = min(max(s.starts[b], 0), s.total);
  n = min(max(s.starts[b + 1], first), s.total) - first;
}

struct ConvArgs {
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* bias;
  uint16_t* state;
  uint16_t* out;
  long x_ts;
  Sequences s;
  int C;
  bool silu;
};
hipError_t launch_conv(const ConvArgs& a, int width, hipStream_t stream);

struct DeltaArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* a;
  const uint16_t* b;
  const float* a_log;
  const float* dt_bias;
  float* state;
  uint16_t* out;
  void* workspace;
  size_t keys;            // where in it the chunks' keys begin
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, a_ts, b_ts;
  Sequences s;
  int Hk, Hv;
  float scale, eps;
  Divisor by_units, by_heads, by_group;   // set at the launch
};
struct DeltaPlan {
  bool chunks;            // in chunks, or token after token
  size_t keys, workspace;
};
constexpr int kChunk = 64;
DeltaPlan delta_plan(int total, int batch, int max_q, int write_cols, int Hk, int Hv, int dk, int dv);
hipError_t launch_delta_chunks(const DeltaArgs& a, int dk, int dv, hipStream_t stream);
hipError_t launch_delta_steps(const DeltaArgs& a, int dk, int dv, hipStream_t stream);

struct SampleArgs {
  const void* logits;
  const float* uniform;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* logprobs;
  void* workspace;
  long row_stride;
  int rows, V, top_k_all, parts;        // parts: workgroups of a row
  float temperature_all, top_p_all, min_p_all;
  bool bf16;
};
int sample_parts(int rows, int V, bool bf16, int top_k);    // top_k: of all rows; 1 where they have their own
size_t sample_workspace(int rows, int parts);
hipError_t launch_sample(const SampleArgs& a, hipStream_t stream);

}  // namespace dec
