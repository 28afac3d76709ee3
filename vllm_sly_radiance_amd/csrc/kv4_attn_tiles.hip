// Attention over the 4-bit paged cache for gfx950, many query rows: prompt chunks.
//
// A workgroup has 32 W rows of one kv head (queries times the query heads that share it) and walks
// over the tokens they see, 128 at a time (64 at D = 256). Its waves turn the codes of later tokens
// into bf16 in LDS, in matrix-operand order, while they work on these, each wave on 32 rows of its own:
//   S^T = K . Q^T     (32 tokens x 32 rows, 16 channels an instruction)
//   O^T += V^T . P^T  (32 channels x 32 rows, 16 tokens an instruction)
// A lane holds one row (lane % 32) throughout, so the softmax needs one exchange, with lane + 32, and
// the registers of S^T are the operand P^T as they are. The order of tokens in an operand is the one
// that they have there: half h of the wave holds tokens 4 h .. 4 h + 3 of each 8.
//
// The matrix cores and the vector units share the work about evenly: at D = 128 a wave's 32 tokens
// take 512 matrix cycles and some 550 vector cycles, half of them 2^x at a quarter of the rate. So
// both go on at once: the scores of the next 32 tokens run under the weights of these 32, the sums
// under the conversion of codes, instruction by instruction.
//
// A batch's row tiles seldom fill the CUs evenly. Whole rounds of them take a workgroup each; the last
// round's are cut along the tokens into as many parts as pay (attn_parts), which attn_join weighs:
// 300 units of 128 rows against 4096 tokens each at D = 256 took 310 us in two rounds of whole
// units, and take 206 and 8 for the join with 44 of them in 5 parts.
//
// 4096 causal tokens, 32 query and 8 kv heads of 128: 138 us, 1000 TFLOP/s of visible products, once the
// card is warm (the first passes 151; a large library product of bf16 matrices reaches 1206). The matrix
// cores are busy 44 % of the cycles, the vector units 48 %. Whole steps pipelined in place of 32 tokens, 2
// to 10 operands read ahead and a second accumulator for the scores were slower or the same; steps of 64
// tokens were 15 % slower (a barrier and a start of the operand reads each). The instance for heads of 128
// spills 2 vector registers, outside of its loop.
#include <utility>

#include "kv4_attn.h"
#include "kv4_attn_shared.h"

namespace kv4 {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kAhead = 3;   // operands read from LDS before their matrix instructions

// LDS-only barrier: what a wave wrote to LDS before it is there for the others; loads from memory
// stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ v16f mfma32(v8bf a, v8bf b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The larger of a lane's value and that of lane ^ 32.
__device__ __forceinline__ float max_halves(float x) { return fmaxf(x, __shfl_xor(x, 32)); }

template <int D, int W>
struct Tiles {
  static constexpr int kRows = 32 * W;
  static constexpr int kTile = D == 256 ? 64 : 128; // tokens of a step
  static constexpr int kSubs = kTile / 32;          // 32 tokens at a time
  static constexpr int kParts = W * kGroup / kTile; // waves that fill a group of 16 tokens
  static constexpr int kLanes = 64 * kParts;
  static constexpr int kKeyUnits = 2 * D / kLanes;  // 4-byte units of key codes a lane converts
  static constexpr int kSteps = D / 16;             // matrix instructions over the channels
  static constexpr int kPlanes = Group<D>::kPlanes;
  // lanes of a group's values: (plane, run, half) x the bytes of a run that lanes share
  static constexpr int kValueUnits = kPlanes * 32;
  static constexpr int kRunBytes = Group<D>::kRunBytes;
  static constexpr int kByteLanes = kLanes / kValueUnits >= kRunBytes ? kRunBytes : kLanes / kValueUnits;
  static constexpr int kBytes = kRunBytes / kByteLanes;   // bytes of a run a lane converts
  static_assert(kKeyUnits >= 2 && kByteLanes >= 1, "tiles");
};

template <int D, int W>
struct Shared {
  static constexpr int kTile = Tiles<D, W>::kTile;
  v4i k[2][kTile / 32][D / 16][64];       // [buffer][32 tokens][16 channels][lane]
  v4i v[2][D / 32][kTile / kGroup][64];   // [buffer][32 channels][16 tokens][lane, in value_slot's order]
  uint8_t nan[2][D / 32][kTile];          // value scales of a step that has NaN blocks
  int has_nan[2];
};

// Where channel c of 32, half h of the tokens, lies among the 64 operands of a matrix instruction. In
// plain order the lanes that write at once, neighbouring runs and halves, would meet in the same LDS
// banks; in this one they do not, nor do those that read at once (lanes 4 i .. 4 i + 3 with the four 16
// + 4 further on or back).
__device__ __forceinline__ int value_slot(int h, int c) {
  const int run = c >> 3;
  return h * 32 + (c ^ ((run & 1) << 2 | (run & 2)) ^ h);
}

// f(0), ..., f(N - 1) with compile-time arguments
template <typename F, int... I>
__device__ __forceinline__ void static_for(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F f) {
  static_for(std::make_integer_sequence<int, N>(), f);
}

// A wave's share of a step's codes, and their way into LDS. Key codes: a lane has kKeyUnits runs of 8
// channels of one token. Value codes: 4 tokens (4 h ..) and 4 more (8 + 4 h ..) of a run of 8
// channels, kBytes of whose bytes are this lane's.
template <int D, int W>
struct Fill {
  using T = Tiles<D, W>;
  using G = Group<D>;
  typedef typename std::conditional<D >= 128, v4i, v2i>::type Vec;
  uint32_t k[T::kKeyUnits];
  uint32_t ks;             // the word that holds the units' key scales (a byte for each 4), from bit ks_bit
  uint32_t key_nan;        // and their tokens' Tokens::nan
  Vec v[2];
  uint32_t vs[2];
  float s[8];              // while they are converted: the tokens' scales, one byte's values
  uint32_t x[8];
  // This lane's places, in bytes: of its keys, their scales, its values and their scales in the group,
  // and in LDS (of a buffer) of its keys and of the two channels of a byte of its values. They are
  // pinned where they are used: 64-bit forms of them would be kept in registers through the loop.
  uint32_t key_at, key_scale_at, ks_bit, value_at, value_scale_at, key_to, even_to, odd_to, nan_to;
  int byte;
  bool has_values;

  __device__ __forceinline__ void place(int grp, int part, int lane) {
    const int l = part * 64 + lane, token = l & 15, run = l >> 4, u = l / T::kByteLanes;
    key_at = G::kKeys + token * (D / 2) + run * (4 * T::kKeyUnits);
    const int scale = token * (D / kBlock) + run * T::kKeyUnits / 4;
    key_scale_at = G::kKeyScales + (scale & ~3), ks_bit = 8 * (scale & 3);
    const int unit = run * T::kKeyUnits, tok = 16 * grp + token;
    key_to = (((tok >> 5) * (D / 16) + (unit >> 1)) * 64 + (unit & 1) * 32 + (tok & 31)) * 16;
    has_values = u < T::kValueUnits;
    byte = l % T::kByteLanes;
    const int h = u & 1, r = (u >> 1) & 15, p = u >> 5, block = D >= 128 ? 4 * p + (r >> 2) : r >> 3;
    value_at = G::kValues + ((p * 4 + h) * 16 + r) * sizeof(Vec);
    value_scale_at = G::kValueScales + block * kGroup + 4 * h;
    const int ch = p * 128 + r * G::kRun + 2 * T::kBytes * byte;
    even_to = ((ch >> 5) * (T::kTile / kGroup) + grp) * 1024 + value_slot(h, ch & 31) * 16;
    odd_to = ((ch >> 5) * (T::kTile / kGroup) + grp) * 1024 + value_slot(h, (ch & 31) + 1) * 16;
    nan_to = block * T::kTile + 16 * grp + 4 * h;
  }

  __device__ __forceinline__ void load_keys(const Tokens& tokens) {
    const uint8_t* group = tokens.group;
    key_nan = tokens.nan;
    const uint8_t* kp = group + (uint32_t)pinned(key_at);
    if constexpr (T::kKeyUnits >= 4) {
#pragma unroll
      for (int i = 0; i < T::kKeyUnits; i += 4) {
        const v4i x = *reinterpret_cast<const v4i*>(kp + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[i + j] = x[j];
      }
    } else {
      static_assert(T::kKeyUnits == 2, "keys");
      const v2i x = *reinterpret_cast<const v2i*>(kp);
      k[0] = x[0], k[1] = x[1];
    }
    // (a word and not the bytes: bytes carried to the next step are masked where they are loaded, with a
    // wait for all that is in flight)
    ks = *reinterpret_cast<const uint32_t*>(group + (uint32_t)pinned(key_scale_at));
  }
  // (lanes without values read those of group byte 0 on: they are not used)
  __device__ __forceinline__ void load_values(const uint8_t* group) {
    const uint8_t* vp = group + (uint32_t)pinned(has_values ? value_at : 0);
    const uint8_t* sp = group + (uint32_t)pinned(has_values ? value_scale_at : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[i] = *reinterpret_cast<const Vec*>(vp + 32 * sizeof(Vec) * i);
      vs[i] = *reinterpret_cast<const uint32_t*>(sp + 8 * i);
    }
  }

  // NaN blocks do not go into the products, where a weight of zero would not hide them: their scales
  // are taken out, and left in LDS for the rows that see them.
  __device__ __forceinline__ void take_out_nan(Shared<D, W>& sh, int buf) {
    const uint32_t nan = has_values ? nan_scales(vs[0]) | nan_scales(vs[1]) : 0;
    if (!__ballot(nan != 0)) return;
    if (!has_values) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t hit = nan_scales(vs[i]);
      *reinterpret_cast<uint32_t*>(&sh.nan[buf][0][0] + nan_to + 8 * i) = hit;
      vs[i] &= ~((hit >> 7) * 0xFFu);
    }
    if (nan) sh.has_nan[buf] = 1;
  }

  // The conversion in slices of some 8 to 16 vector instructions, to go between matrix instructions.
  static constexpr int kSlices = T::kKeyUnits + 1 + 3 * T::kBytes;
  template <int I>
  __device__ __forceinline__ void slice(Shared<D, W>& sh, int kbuf, int vbuf) {
    if constexpr (I < T::kKeyUnits) {
      // units I and I + 1 are the two halves of an instruction's channels
      uint8_t* to = reinterpret_cast<uint8_t*>(&sh.k[kbuf][0][0][0]) + pinned(key_to);
      const uint32_t e = ((ks | key_nan) >> (ks_bit + 8 * (I / 4))) & 0xFFu;
      const v4i y = __builtin_bit_cast(v4i, expand8(k[I], stored_scale(e)));
      *reinterpret_cast<v4i*>(to + (I >> 1) * 1024 + (I & 1) * 512) = y;
    } else if constexpr (I == T::kKeyUnits) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = scale_of((vs[i >> 2] >> (8 * (i & 3))) & 0xFFu);
    } else {
      constexpr int B = (I - T::kKeyUnits - 1) / 3, what = (I - T::kKeyUnits - 1) % 3;
      if constexpr (what == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t w = (uint32_t)v[i >> 2][D >= 128 ? i & 3 : (i & 3) >> 1];
          if constexpr (D == 64) w >>= 16 * (i & 1);
          if constexpr (T::kByteLanes > 1) w >>= 8 * T::kBytes * byte;
          x[i] = codes_bf16x2<B>(w, s[i]);
        }
      } else {
        const v4i y = what == 1 ? v4i{halves_lo(x[0], x[1]), halves_lo(x[2], x[3]),
                                      halves_lo(x[4], x[5]), halves_lo(x[6], x[7])}
                                : v4i{halves_hi(x[0], x[1]), halves_hi(x[2], x[3]),
                                      halves_hi(x[4], x[5]), halves_hi(x[6], x[7])};
        // byte B of a run is channels 2 B and 2 B + 1 of it; value_slot's order is an exclusive or
        uint8_t* base = reinterpret_cast<uint8_t*>(&sh.v[vbuf][0][0][0]);
        const uint32_t to = pinned(what == 1 ? even_to : odd_to) ^ (2 * B * 16);
        if (has_values) *reinterpret_cast<v4i*>(base + to) = y;
      }
    }
  }
  // slices [A, B)
  template <int A, int B>
  __device__ __forceinline__ void slices(Shared<D, W>& sh, int kbuf, int vbuf) {
    static_for<B - A>([&](auto i) { slice<A + decltype(i)::value>(sh, kbuf, vbuf); });
  }
};

// Row tiles of sequence i: as many as its rows fill where it has more than attn_rows takes; a bad one has
// one, which writes its NaN.
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int tile_rows, int i) {
  if (i >= a.batch) return 0;
  const Sequence s = sequence(a, i);
  const int R = s.bad ? 0 : s.n * a.group;
  return s.bad ? 1 : R > a.few_rows ? ceil_div(R, tile_rows) : 0;
}

// The x-th row tile from the end of the batch's.
struct Place { int b, tile; };
__device__ __forceinline__ Place find_tile(const AttnArgs& a, int tile_rows, int x, int lane) {
  int left = x;
  for (int i0 = (a.batch - 1) & ~63; i0 >= 0; i0 -= 64) {
    const int n = tiles_of(a, tile_rows, i0 + 63 - lane);   // lanes in descending order
    const int upto = wave_scan(n);
    const uint64_t here = __ballot(left >= upto - n && left < upto);
    if (here) {
      const int k = __builtin_ctzll(here);
      return {i0 + 63 - k, __builtin_amdgcn_readlane(upto, k) - 1 - left};
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0};
}

// What workgroup x does: one of `parts` parts of the tokens of unit `unit` (row tile and kv head), whose
// partial results are those of entry `entry`. Units that fill whole rounds of the CUs are done by a
// workgroup each; those of the last round, which would leave CUs idle, in parts.
struct Work { int unit, part, parts, entry; };
__device__ __forceinline__ Work find_work(const AttnArgs& a, int tile_rows, int x, int lane) {
  if (!a.entries) return {x, 0, 1, 0};
  int tiles = 0;
  for (int i0 = 0; i0 < a.batch; i0 += 64)
    tiles += __builtin_amdgcn_readlane(wave_scan(tiles_of(a, tile_rows, i0 + lane)), 63);
  const int units = tiles * a.Hkv, rest = units % kCUs, first = units - rest;
  const int parts = attn_parts(rest, a.span, a.entries);
  // attn_join looks at the entries that there may be. Those past the batch's have nothing for it, nor have
  // those whose workgroup was not launched, where starts that go back make more units than were planned for
  // (asked here only: `rest` chosen by a.units cost 4 us of 225 with 300 units at D = 256).
  if (x < a.entries && x < kCUs && threadIdx.x == 0 && (x >= rest || first + x >= a.units + a.entries))
    meta(a, tile_rows, a.d, x)[0] = 0;
  if (x < first) return {x, 0, 1, -1};
  const int y = x - first, part = rest ? y / rest : parts;
  if (part >= parts) return {units, 0, 1, -1};
  return {first + y - part * rest, part, parts, y - part * rest};
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, W / 4) void attn_tiles(AttnArgs a) {
  using T = Tiles<D, W>;
  using G = Group<D>;
  constexpr int KS = T::kSteps, CT = D / 32, kTile = T::kTile;
  __shared__ Shared<D, W> sh;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // Units [tiles of the batch, the last first][kv heads]. A sequence's last tiles, which see most tokens,
  // begin first; and where the kv heads are a multiple of 8 a head's keys and values stay in one
  // die's L2.
  const Work work = find_work(a, T::kRows, blockIdx.x, lane);
  const int x = a.by_heads(work.unit), h = work.unit - x * a.Hkv;
  const Place at = find_tile(a, T::kRows, x, lane);
  if (at.b < 0) return;
  const int b = at.b, tile = at.tile;
  const Sequence s = sequence_uniform(a, b);
  if (a.entries && work.entry >= 0 && work.part == 0 && tid == 0) {
    int* mt = meta(a, T::kRows, D, work.entry);
    mt[0] = s.bad ? 0 : work.parts - 1;
    mt[1] = b, mt[2] = tile * a.Hkv + h, mt[3] = work.entry * work.parts;
  }
  if (s.bad) {
    nan_rows<D>(a, s, h * a.group, a.group);
    return;
  }
  const int R = s.n * a.group, r0 = tile * T::kRows;
  const Span all = query_span(a, s, a.by_group(r0), a.by_group(min(r0 + T::kRows, R) - 1));

  // this wave's rows
  const int w0 = r0 + 32 * wave;
  const int row = min(w0 + (lane & 31), R - 1), qi = a.by_group(row);
  const Span mine = query_span(a, s, a.by_group(min(w0, R - 1)), a.by_group(min(w0 + 32, R) - 1));
  const int place = s.len - s.n + qi;
  const int hi = a.causal ? min(place + 1, s.len) : s.len;
  const int lo = first_seen(a, place);
  v8bf q[KS];
  {
    const uint16_t* src = a.q + (size_t)(s.q0 + qi) * a.q_ts +
                          (size_t)(h * a.group + row - qi * a.group) * a.q_hs + 8 * half;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      q[k] = __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(src + 16 * k));
  }

  // filling: wave w has a share (part) of the 16 tokens of group grp of each step
  const int grp = wave / T::kParts;
  const int* table = a.pages_of + (size_t)b * a.table_stride;
  const uint8_t* head_base = a.cache + (size_t)(h << (a.page_shift - 4)) * G::kBytes;
  const int group_mask = (1 << (a.page_shift - 4)) - 1;
  // this workgroup's part of the tokens, in steps
  const int share = ceil_div(ceil_div(max(all.hi - all.lo, 0), kTile), work.parts) * kTile;
  const int t0 = all.lo + work.part * share, t1 = min(all.hi, t0 + share);
  const int last_page = (t1 - 1) >> a.page_shift;
  // The numbers of 128 pages from page_base on, a lane each of two registers: a step's is read from them
  // without a wait. (A scalar load would share its counter with the LDS reads and stall them.)
  auto pages_from = [&](int first) { return table[min(first + lane, last_page)]; };
  int page_base = 0, pages_now = 0, pages_next = 0;
  auto group_at = [&](int t) {
    t += 16 * grp;
    const int e = min(t >> a.page_shift, last_page);
    if (e >= page_base + 64) {
      page_base += 64;
      pages_now = pages_next;
      pages_next = pages_from(page_base + 64);
    }
    return tokens_at(a, head_base, __builtin_amdgcn_readlane(pages_now, e - page_base),
                     (t >> 4) & group_mask, G::kBytes);
  };

  const float c = a.scale * 1.44269504088896340736f;
  const float slack = 8.0f / c;
  float m = -INFINITY, l = 0.0f;
  v16f o[CT], sc[2];                      // scores of the step's first 32 tokens, and of the others
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;

  // Filling runs ahead by as much as the buffers allow: a step writes the first 32 keys of the step
  // after the next, and the other 32 keys and the values of the next.
  const int key_ahead = grp < 2 ? 2 : 1;
  const int value_lane = value_slot(half, lane & 31);
  Fill<D, W> fill;
  fill.place(grp, wave % T::kParts, lane);
  Tokens keys_from = {};                  // whose keys are in `fill`
  if (tid == 0) sh.has_nan[0] = sh.has_nan[1] = 0;
  for (int i = tid; i < 2 * CT * kTile; i += 64 * W) (&sh.nan[0][0][0])[i] = 0;
  lds_barrier();
  if (t0 < t1) {
    page_base = t0 >> a.page_shift;
    pages_now = pages_from(page_base), pages_next = pages_from(page_base + 64);
    const Tokens g0 = group_at(t0);
    const Tokens g1 = group_at(t0 + kTile);
    fill.load_keys(g0);
    fill.load_values(g0.group);
    fill.take_out_nan(sh, 0);
    fill.template slices<0, Fill<D, W>::kSlices>(sh, 0, 0);
    if (grp < 2) {
      fill.load_keys(g1);
      fill.template slices<0, T::kKeyUnits>(sh, 1, 0);
      keys_from = group_at(t0 + 2 * kTile);
    } else {
      keys_from = g1;
    }
    fill.load_keys(keys_from);
    fill.load_values(g1.group);
    lds_barrier();
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[0][j] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      sc[0] = mfma32(__builtin_bit_cast(v8bf, sh.k[0][0][k][lane]), q[k], sc[0]);
  }
  // The queries are here: without this the compiler waits for them inside the loop, each step, and with
  // them for the loads just asked for.
  __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt(0)
  int buf = 0;                            // of step t; buf ^ 1 of step t + 1
  for (int t = t0; t < t1; t += kTile, buf ^= 1) {
    // all have written what this step reads, and read what it overwrites
    lds_barrier();
    const int nan_here = sh.has_nan[buf];
    // Operands in the order of their use, read kAhead instructions before it: the keys of the step's
    // other 32 tokens, the values of its first, the first 32 keys of the next step, the other values.
    constexpr int U = T::kSubs, NK = KS, NV = 2 * CT, N = U * (NK + NV);
    auto operand = [&](auto i) {
      constexpr int n = decltype(i)::value % (NK + NV), u = decltype(i)::value / (NK + NV);
      if constexpr (n < NK) return sh.k[u + 1 == U ? buf ^ 1 : buf][(u + 1) % U][n][lane];
      else return sh.v[buf][(n - NK) % CT][2 * u + (n - NK) / CT][value_lane];
    };
    v4i ring[kAhead];
    static_for<kAhead>([&](auto i) { ring[decltype(i)::value] = operand(i); });
    auto next_operand = [&](auto i) {
      constexpr int n = decltype(i)::value;
      const v8bf y = __builtin_bit_cast(v8bf, ring[n % kAhead]);
      if constexpr (n + kAhead < N) ring[n % kAhead] = operand(std::integral_constant<int, n + kAhead>());
      return y;
    };
    static_for<U>([&](auto part) {
      constexpr int u = decltype(part)::value, first = u * (NK + NV), x = u & 1;
      if (t + 32 * u + 32 > mine.all_hi || t + 32 * u < mine.all_lo) {                          // tokens that some row does not see
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int tok = t + 32 * u + 8 * (j >> 2) + 4 * half + (j & 3);
          if (tok >= hi || tok < lo) sc[x][j] = -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[x][j]);
      if (__ballot(mx > m + slack)) {
        const float mn = fmaxf(m, max_halves(mx));
        const float alpha = mn == m ? 1.0f : exp2_raw((m - mn) * c);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[i][j] *= alpha;
      }
      const float sub = m == -INFINITY ? 0.0f : m * c;
      if constexpr (u == U / 2) fill.take_out_nan(sh, buf ^ 1);
      __builtin_amdgcn_sched_barrier(0);

      // the scores of the next 32 tokens, and between them the weights of these
      uint32_t p[8];
      float e0 = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[x ^ 1][j] = 0.0f;
      static_for<NK>([&](auto i) {
        constexpr int n = decltype(i)::value;
        sc[x ^ 1] = mfma32(next_operand(std::integral_constant<int, first + n>()), q[n], sc[x ^ 1]);
        static_for<16 * (n + 1) / NK - 16 * n / NK>([&](auto k) {
          constexpr int j = 16 * n / NK + decltype(k)::value;
          const float e = exp2_raw(fmaf(sc[x][j], c, -sub));
          l += e;
          if constexpr (j & 1) p[j >> 1] = bf16x2(e0, e);
          else e0 = e;
        });
      });
      // the sums over these 32 tokens, and between them codes on their way into LDS
      static_for<NV>([&](auto i) {
        constexpr int n = decltype(i)::value, g = n / CT, S = Fill<D, W>::kSlices;
        const v4i pd = {(int)p[4 * g], (int)p[4 * g + 1], (int)p[4 * g + 2], (int)p[4 * g + 3]};
        o[n % CT] = mfma32(next_operand(std::integral_constant<int, first + NK + n>()),
                           __builtin_bit_cast(v8bf, pd), o[n % CT]);
        // the keys under the first half of the sums, the values under the second
        constexpr int H = U / 2 * NV, at = u % (U / 2) * NV + n;
        constexpr int S0 = u < U / 2 ? 0 : T::kKeyUnits, S1 = u < U / 2 ? T::kKeyUnits : S;
        fill.template slices<S0 + at * (S1 - S0) / H, S0 + (at + 1) * (S1 - S0) / H>(
            sh, grp < 2 ? buf : buf ^ 1, buf ^ 1);
      });
    });
    const uint8_t* values_from = (grp < 2 ? keys_from : group_at(t + 2 * kTile)).group;
    keys_from = group_at(t + (key_ahead + 1) * kTile);
    fill.load_keys(keys_from);             // needed first
    fill.load_values(values_from);
    if (nan_here) {
      // Rows that see a token with a NaN block: its 32 channels are NaN. 2^127 for the block times
      // 2^127 for the row that sees it is infinite; the same once more with the other sign is NaN.
      // (Products, because the accumulators stay where the matrix instructions have them.)
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll 1
        for (int g = 0; g < kTile / kGroup; ++g) {
          float mark[8], sees[8];
          int any = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int tok = 16 * g + 8 * (j >> 2) + 4 * half + (j & 3);
            const int hit = sh.nan[buf][i][tok];
            any |= hit;
            mark[j] = hit ? 0x1p127f : 0.0f;
            sees[j] = t + tok < hi && t + tok >= lo ? 0x1p127f : 0.0f;
          }
          if (!__ballot(any != 0)) continue;
          const v8bf x = pack8bf(mark), y = pack8bf(sees);
          o[i] = mfma32(x, y, o[i]);
#pragma unroll
          for (int j = 0; j < 8; ++j) mark[j] = -mark[j];
          o[i] = mfma32(pack8bf(mark), y, o[i]);
        }
      lds_barrier();                       // all have read the marks: they go for the next use
      if (tid == 0) sh.has_nan[buf] = 0;
      for (int i = tid; i < CT * kTile; i += 64 * W) sh.nan[buf][i / kTile][i % kTile] = 0;
    }
  }

  l += __shfl_xor(l, 32);
  if (w0 + (lane & 31) >= R) return;
  if (work.parts == 1 && hi <= max(lo, 0)) l = INFINITY;
  uint16_t* out = out_row(a, D, s.q0, h, row);
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float y[4] = {o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
      const int ch = 32 * i + 8 * g + 4 * half;
      if (work.parts == 1)
        store_row<4>(out + ch, y, l);
      else
        store_part<4>(a, T::kRows, D, work.entry * work.parts + work.part, row - r0, ch, y, m * c, l);
    }
}

template <int D, int W>
hipError_t launch(AttnArgs a, hipStream_t stream) {
  constexpr int kRows = Tiles<D, W>::kRows;
  a.by_group = divisor(a.group), a.by_heads = divisor(a.Hkv);
  a.d = D, a.runs = (a.entries + 1) / 2;
  attn_tiles<D, W><<<a.units + a.entries, 64 * W, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (!a.entries) return hipSuccess;
  a.by_parts = true;
  const int entries = a.entries < kCUs ? a.entries : kCUs - 1;
  return launch_attn_join(a, D, kRows, entries < a.units ? entries : a.units, stream);
}

}  // namespace

int attn_tile_rows(int d) { return d == 256 ? Tiles<256, 4>::kRows : Tiles<128, 8>::kRows; }

hipError_t launch_attn_tiles(const AttnArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch<64, 8>(a, stream)
                 : d == 128 ? launch<128, 8>(a, stream) : launch<256, 4>(a, stream);
}

}  // namespace kv4
