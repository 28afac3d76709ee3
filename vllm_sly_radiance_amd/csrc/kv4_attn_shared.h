// Device helpers of the attention kernels over the 4-bit cache. Not part of the C ABI.
#pragma once
#include <type_traits>

#include "kv4_internal.h"

namespace kv4 {

// Waves of a workgroup of attn_rows, and waves a SIMD is to hold (registers allow no more).
constexpr int kRunWaves = 4;                                          // sharing the batch's tokens
constexpr int attn_whole_waves(int rf) { return rf <= 2 ? 8 : 4; }    // a workgroup a unit
constexpr int attn_waves(int d, int rf) { return d * rf <= 128 ? 4 : d * rf <= 256 || d < 256 ? 2 : 1; }

__device__ __forceinline__ v4f mfma16(v8bf a, v8bf b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A scalar load: the address is the same in every lane, and nothing writes there while the kernel
// runs.
__device__ __forceinline__ int scalar_load(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(uintptr_t)p;
}

// x, which the compiler computes with from here on and not earlier.
template <typename I>
__device__ __forceinline__ I pinned(I x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A value that is the same in every lane, as a scalar.
__device__ __forceinline__ long uniform(long x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)x);
  return ((long)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | lo;
}

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// Inclusive scan over the wave: shifts inside rows of 16 lanes, then the rows' last lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);   // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);   // row_bcast:15, rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);   // row_bcast:31, rows 2 and 3
  return x;
}

// A sequence of the batch: its tokens, its first query row, its queries. Sizes that do not fit what
// the launch was planned for make it bad: its rows are NaN.
struct Sequence { int len, q0, n; bool bad; };
__device__ __forceinline__ bool misfit(const AttnArgs& a, const Sequence& s) {
  const long pages = ((long)s.len + (1 << a.page_shift) - 1) >> a.page_shift;
  return s.len < 0 || s.len > a.max_len || pages > a.table_cols || s.q0 < 0 || s.n < 0 ||
         s.n > a.max_q || s.q0 > a.total - s.n;
}
__device__ __forceinline__ Sequence sequence(const AttnArgs& a, int b) {
  Sequence s;
  s.len = a.lens[b];
  s.q0 = a.starts[b];
  s.n = a.starts[b + 1] - s.q0;
  s.bad = misfit(a, s);
  return s;
}
// the same of a b that is the same in every lane
__device__ __forceinline__ Sequence sequence_uniform(const AttnArgs& a, int b) {
  Sequence s;
  s.len = scalar_load(a.lens + b);
  s.q0 = scalar_load(a.starts + b);
  s.n = scalar_load(a.starts + b + 1) - s.q0;
  s.bad = misfit(a, s);
  return s;
}

// A group of 16 tokens. Those of a page number outside the cache are read from page 0, and `nan` (all ones;
// 0 for others), set in the words of their key scales, makes their scores NaN: the masks keep that from the
// rows that do not see them.
struct Tokens { const uint8_t* group; uint32_t nan; };
__device__ __forceinline__ Tokens tokens_at(const AttnArgs& a, const uint8_t* head_base, int page, int group,
                                            int group_bytes) {
  const bool ok = (uint32_t)page < (uint32_t)a.pages;
  return {head_base + (uint64_t)(uint32_t)(ok ? page : 0) * (uint32_t)a.page_stride +
              (uint32_t)group * (uint32_t)group_bytes, ok ? 0u : ~0u};
}

// The first token that a query at `place` sees; at most 0: no bound. A query before the sequence (more
// queries than tokens) counts as at its start, where a window ends before the tokens too: its own place less
// a window as large as an int would wrap, to a start far behind the pages.
__device__ __forceinline__ int first_seen(const AttnArgs& a, int place) {
  return a.window > 0 ? max(place, 0) - a.window + 1 : 0;
}

// Whether a query at `place` of a sequence of len tokens sees any.
__device__ __forceinline__ bool sees_any(const AttnArgs& a, int len, int place) {
  return (a.causal ? min(place + 1, len) : len) > max(first_seen(a, place), 0);
}

// Tokens [lo, hi) that the queries first .. last of a sequence see between them (lo rounded down to a
// step), and [all_lo, all_hi) that each of them sees.
struct Span { int lo, hi, all_lo, all_hi; };
__device__ __forceinline__ Span query_span(const AttnArgs& a, const Sequence& s, int first, int last) {
  const int p0 = s.len - s.n + first, p1 = s.len - s.n + last;
  Span x;
  x.hi = a.causal ? min(s.len, max(p1 + 1, 0)) : s.len;
  x.all_hi = a.causal ? min(s.len, p0 + 1) : s.len;
  x.lo = max(first_seen(a, p0), 0) & ~31;
  x.all_lo = first_seen(a, p1);
  return x;
}

// NaN to every output row of a bad sequence that lies in the output, for `heads` heads from h0.
template <int D>
__device__ __forceinline__ void nan_rows(const AttnArgs& a, const Sequence& s, int h0, int heads) {
  const long first = max(s.q0, 0);
  const long last = min((long)s.q0 + s.n, (long)a.total);
  for (long i = first * heads * D + threadIdx.x; i < last * heads * D; i += blockDim.x) {
    const long row = i / (heads * D), at = i % (heads * D);
    a.out[(row * a.Hq + h0) * D + at] = 0x7FC0;
  }
}

// The output of row `row` (queries times the heads of a group) of a sequence's kv head.
__device__ __forceinline__ uint16_t* out_row(const AttnArgs& a, int D, int q0, int h, int row) {
  const int qi = a.by_group(row);
  return a.out + ((size_t)(q0 + qi) * a.Hq + h * a.group + row - qi * a.group) * D;
}

// 8 codes as a bf16 operand.
__device__ __forceinline__ v8bf expand8(uint32_t codes, float scale) {
  const v4i r = {(int)codes_bf16x2<0>(codes, scale), (int)codes_bf16x2<1>(codes, scale),
                 (int)codes_bf16x2<2>(codes, scale), (int)codes_bf16x2<3>(codes, scale)};
  return __builtin_bit_cast(v8bf, r);
}

__device__ __forceinline__ v8bf pack8bf(const float e[8]) {
  const v4i r = {(int)bf16x2(e[0], e[1]), (int)bf16x2(e[2], e[3]), (int)bf16x2(e[4], e[5]),
                 (int)bf16x2(e[6], e[7])};
  return __builtin_bit_cast(v8bf, r);
}

// Bit 7 of each of four scale bytes above 252, which read as NaN.
__device__ __forceinline__ uint32_t nan_scales(uint32_t four) {
  return ((four & 0x7F7F7F7Fu) + 0x03030303u) & four & 0x80808080u;
}

// The low (high) halves of two dwords, the first one's below.
__device__ __forceinline__ int halves_lo(uint32_t x, uint32_t y) {
  return (int)__builtin_amdgcn_perm(y, x, 0x05040100u);
}
__device__ __forceinline__ int halves_hi(uint32_t x, uint32_t y) {
  return (int)__builtin_amdgcn_perm(y, x, 0x07060302u);
}

// Byte B (channels 2 B, 2 B + 1 of the run) of 4 + 4 tokens' codes as the two channels' operands.
template <int B, typename F>
__device__ __forceinline__ void value_pair(v8bf& even, v8bf& odd, F codes, const float s[8]) {
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = codes(i, s[i], std::integral_constant<int, B>());
  const v4i lo = {halves_lo(x[0], x[1]), halves_lo(x[2], x[3]), halves_lo(x[4], x[5]),
                  halves_lo(x[6], x[7])};
  const v4i hi = {halves_hi(x[0], x[1]), halves_hi(x[2], x[3]), halves_hi(x[4], x[5]),
                  halves_hi(x[6], x[7])};
  even = __builtin_bit_cast(v8bf, lo);
  odd = __builtin_bit_cast(v8bf, hi);
}

// A run's channels as operands over the 8 tokens of a lane (4 g + i of two groups of 16), two
// channels at a time: use(index of the pair, channel 2 x index, the one after).
template <int D, typename Vec, typename Use>
__device__ __forceinline__ void each_value_pair(Vec v0, uint32_t s0, Vec v1, uint32_t s1, Use use) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = scale_of((s0 >> (8 * i)) & 0xFFu);
    s[4 + i] = scale_of((s1 >> (8 * i)) & 0xFFu);
  }
  auto codes = [&](int i, float sc, auto b) {
    constexpr int B = decltype(b)::value;
    if constexpr (D >= 128) {         // dword i: token i's 4 bytes
      return codes_bf16x2<B>((uint32_t)(i < 4 ? v0[i] : v1[i - 4]), sc);
    } else {                          // dword i / 2: tokens i, i + 1, 2 bytes each
      const uint32_t w = (uint32_t)(i < 4 ? v0[i >> 1] : v1[(i - 4) >> 1]);
      return i & 1 ? codes_bf16x2<(B + 2) % 4>(w, sc) : codes_bf16x2<B>(w, sc);
    }
  };
  v8bf even, odd;
  value_pair<0>(even, odd, codes, s);
  use(std::integral_constant<int, 0>(), even, odd);
  value_pair<1>(even, odd, codes, s);
  use(std::integral_constant<int, 1>(), even, odd);
  if constexpr (D >= 128) {
    value_pair<2>(even, odd, codes, s);
    use(std::integral_constant<int, 2>(), even, odd);
    value_pair<3>(even, odd, codes, s);
    use(std::integral_constant<int, 3>(), even, odd);
  }
}

// C consecutive channels of an output row: y / sum in bf16. A query that sees nothing has y = 0 and is given
// an infinite sum, for zeros; one whose scores are all -infinity has y = 0 and sum = 0, for NaN.
template <int C>
__device__ __forceinline__ void store_row(uint16_t* out, const float y[C], float sum) {
  const float inv = 1.0f / sum;
  float z[C];
#pragma unroll
  for (int i = 0; i < C; ++i) z[i] = y[i] * inv;
  if constexpr (C == 1) {
    *out = (uint16_t)bf16x2(z[0], 0.0f);
  } else {
    uint32_t w[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i) w[i] = bf16x2(z[2 * i], z[2 * i + 1]);
    __builtin_memcpy(__builtin_assume_aligned(out, 2 * C < 16 ? 2 * C : 16), w, 2 * C);
  }
}

// Workspace of attn_rows: partial results fp32 [2 runs][tile rows][D], [2 runs][tile rows][2] with
// the row's maximum (in units of log2) and sum, and int [runs][4]: what attn_join is told (of a unit,
// by its index b * units + unit, or of the one that begins in a run). attn_tiles' has the same parts,
// a partial result for each part of each entry (2 runs of them at least), and int [256][4], by entry.
__device__ __forceinline__ float* part_row(const AttnArgs& a, int tile_rows, int D, int slot,
                                           int row) {
  return a.part + ((size_t)slot * tile_rows + row) * D;
}
__device__ __forceinline__ float* part_stat(const AttnArgs& a, int tile_rows, int D, int slot,
                                            int row) {
  return a.part + (size_t)2 * a.runs * tile_rows * D + ((size_t)slot * tile_rows + row) * 2;
}
__device__ __forceinline__ int* meta(const AttnArgs& a, int tile_rows, int D, int entry) {
  return reinterpret_cast<int*>(a.part + (size_t)2 * a.runs * tile_rows * (D + 2)) + 4 * entry;
}
template <int C>
__device__ __forceinline__ void store_part(const AttnArgs& a, int tile_rows, int D, int slot,
                                           int row, int ch, const float y[C], float top,
                                           float sum) {
  float* o = part_row(a, tile_rows, D, slot, row) + ch;
#pragma unroll
  for (int i = 0; i < C; i += 4)
    *reinterpret_cast<v4f*>(o + i) = v4f{y[i], y[i + 1], y[i + 2], y[i + 3]};
  if (ch == 0) {
    float* st = part_stat(a, tile_rows, D, slot, row);
    st[0] = top, st[1] = sum;
  }
}

}  // namespace kv4
