// Internals shared by the 4-bit cache and attention kernels for gfx950 (CDNA4). Not part of the C
// ABI; the cache's layout is described in kv4_attn.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace kv4 {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int kGroup = 16;   // tokens of a group
constexpr int kBlock = 32;   // channels of a scale byte

// Byte offsets inside a group of one head of D channels, and the value layout's parameters.
template <int D>
struct Group {
  static constexpr int kPlanes = D >= 128 ? D / 128 : 1;
  static constexpr int kRun = D >= 128 ? 8 : 4;       // channels of a run
  static constexpr int kRunBytes = kRun / 2;
  static constexpr int kKeys = 0;
  static constexpr int kValues = 8 * D;
  static constexpr int kKeyScales = 16 * D;
  static constexpr int kValueScales = 16 * D + D / 2;
  static constexpr int kBytes = 17 * D;
};

__host__ __device__ constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

__device__ __forceinline__ float bits_f32(uint32_t u) { return __uint_as_float(u); }
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// Two fp32 rounded to bf16 (nearest even; v_cvt_pk_bf16_f32), the first in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2bf));
}

// Byte B of four bytes of codes as two bf16, times the scale (its exponent is what the instruction
// takes, so 255 gives NaN and 0 gives 2^-127; every code and scale of the cache is exact in bf16).
template <int B>
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }
// The same with bytes above 252, which scale_byte never gives, as 255: with 253 and 254 some codes pass the
// range of bf16, and an infinite value would reach rows that do not see it through a weight of zero.
__device__ __forceinline__ float stored_scale(uint32_t e) { return scale_of(e > 252u ? 255u : e); }

// A block's scale byte from the largest magnitude's bits: the smallest exponent with amax <= 7 x
// scale. Adding 0x1FFFFF carries into the exponent exactly where the mantissa is above 1.75.
// 252 at most: 6 x 2^125 is the largest of bf16's range; 255 for what is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return 255u;
  const int e = (int)((amax_bits + 0x1FFFFFu) >> 23) - 2;
  return (uint32_t)min(max(e, 1), 252);
}

// Eight fp32 as e2m1 codes in their block's scale (round to nearest even, saturating at 6: what
// v_cvt_scalef32_pk_fp4_f32 does), channel 0 in the lowest nibble. A NaN block's codes are 0.
__device__ __forceinline__ uint32_t codes8(const float y[8], uint32_t e) {
  if (e == 255u) return 0u;
  const float s = scale_of(e);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], s, 3);
  return r;
}

// Division of 0 <= n < 2^31 by a divisor that the host knows: a multiplication by m =
// floor(2^(31 + s) / d) + 1, s = ceil(log2 d), whose error m d - 2^(31 + s) <= d <= 2^s stays below
// what moves a quotient. The integer division in its place is some 40 dependent instructions, and
// several stood before a workgroup's first loads.
struct Divisor {
  int d;
  uint32_t m;
  int shift;              // s - 1
  __device__ __forceinline__ int operator()(int n) const {
    return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> shift);
  }
};
inline Divisor divisor(int d) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  return {d, d == 1 ? 0u : (uint32_t)(((uint64_t)1 << (31 + s)) / (uint64_t)d + 1), s - 1};
}

// ---- arguments of the launchers -----------------------------------------------------------------
struct Heads {            // bf16 [T][heads][d] with unit channel stride
  const uint16_t* p;
  long ts, hs;            // token and head strides, elements
};

struct RopeArgs {
  Heads q, k, v;          // v.p null: k goes to k_out instead of the cache
  const uint16_t* qw;     // bf16 [d], or null: no norm
  const uint16_t* kw;
  const void* table;      // fp32 or bf16 [rows][rot]
  const void* pos;        // int64 or int32 [axes][T]
  const int* axis;        // [rot / 2], or null
  uint16_t* q_out;
  uint16_t* k_out;
  uint8_t* cache;
  const int64_t* slots;
  long rows, pos_stride, pages, page_stride;
  int page_shift, rot, axes, T, Hq, Hkv, flags;
  float eps;
};
hipError_t launch_rope(const RopeArgs& a, int d, hipStream_t stream);

struct GatherArgs {
  const uint8_t* cache;
  const int64_t* slots;
  uint16_t* k;
  uint16_t* v;
  long pages, page_stride;
  int page_shift, T, H;   // T * H < 2^31
  Divisor by_heads;       // of H, set at the launch
};
hipError_t launch_gather(const GatherArgs& a, int d, hipStream_t stream);

constexpr int kMovePairs = 448;   // pairs of one launch: 3584 bytes of its arguments
struct MoveArgs {
  uint8_t* cache;
  long layer_stride, page_stride;
  size_t page_bytes;
  int* tables;
  long table_stride;
  int layers, table_rows, table_cols;
};
// pairs: n <= kMovePairs of them (src, dst), sorted by src
hipError_t launch_move(const MoveArgs& a, const int* pairs, int n, hipStream_t stream);

struct AttnArgs {
  const uint16_t* q;
  const uint8_t* cache;
  const int* pages_of;    // page table
  const int* lens;
  const int* starts;
  uint16_t* out;
  float* part;            // partial results, or null
  long q_ts, q_hs, page_stride, pages, table_stride;
  int page_shift, table_cols, total, batch, max_q, max_len, Hq, Hkv, group, window;   // group: Hq / Hkv
  float scale;
  bool causal;
  int fragments;          // row fragments of attn_rows' workgroups
  int runs;               // workgroups that share the batch's tokens; 0: one a unit
  int few_rows;           // attn_rows has the sequences of at most so many rows, attn_tiles the
                          // others; 0: one of them has all
  // set at the launch: row tiles of a sequence at most, where runs is 0; units of a sequence at most
  // (attn_tiles: of the batch, from the plan), and whether attn_join goes by units (there are no more of
  // them than runs) or by runs
  int tiles, units;
  bool by_unit;
  // attn_tiles: partial results that the workspace holds (0: no unit is done in parts), tokens that a
  // row tile sees at most; the head size; and, for attn_join, that partial results lie by entry and part
  int entries, span, d;
  bool by_parts;
  Divisor by_group, by_heads, by_runs;   // of Hq / Hkv, Hkv, runs
};
constexpr int kCUs = 256;

// Into how many parts of their tokens the `rest` < 256 units of attn_tiles' last round are cut, at most
// `entries` in all. Counted in the time of a unit's token: the parts' rounds, with 140 for a
// workgroup's start and end, and 2 for each partial result's way through memory.
__host__ __device__ inline int attn_parts(int rest, int span, int entries) {
  int best = 1, least = span + 140;
#pragma unroll
  for (int s = 2; s <= 16; ++s) {       // (unrolled, the divisions are multiplications)
    const int cost = (rest * s + kCUs - 1) / kCUs * (span / s + 140) + 2 * rest * s;
    if (rest * s <= entries && cost < least) least = cost, best = s;
  }
  return best;
}

// What serves a call (attn_tiles, attn_rows or both), and the workspace that takes: attn_tiles' first.
struct AttnPlan {
  bool tiles, rows;
  int fragments, runs, few_rows;
  int units, entries, span;             // of attn_tiles; units: at most
  size_t tiles_workspace, workspace;
  long work;                            // granules of attn_rows and starts of its units, where runs share them
  long threads;                         // of the largest launch
};
AttnPlan attn_plan(int total, int batch, int max_q, int max_len, int Hq, int Hkv, int d, int window);
int attn_tile_rows(int d);          // rows of a workgroup of attn_tiles
hipError_t launch_attn_rows(const AttnArgs& a, int d, hipStream_t stream);
hipError_t launch_attn_tiles(const AttnArgs& a, int d, hipStream_t stream);
hipError_t launch_attn_join(const AttnArgs& a, int d, int tile_rows, int entries, hipStream_t stream);

}  // namespace kv4
