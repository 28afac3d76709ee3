// Attention over the 4-bit paged cache for gfx950, few query rows: decode, speculative verify.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c s_j - m),  s_j = q . k_j,  c = scale * log2(e)
//
// The rows of one kv head are its sequence's queries times the query heads that share it; a
// workgroup has 16 * RF of them and a run of the cached tokens, its W waves 32 tokens at a time in
// turn. Keys and values are read once, straight into registers in matrix-operand order:
//   S^T = K . Q^T   (16 tokens x 16 rows): lane (g = l / 16, r = l % 16) holds token r, one block of
//                   32 channels per instruction group; its 16 bytes of codes and one scale.
//   O^T = V^T . P^T (16 channels x 16 rows over 32 tokens): the scores' registers are already the
//                   P^T operand (tokens 4 g + i of both groups of 16), and the value layout gives a
//                   lane the same 8 tokens of the 8 channels of run r.
// Codes become bf16 by v_cvt_scalef32_pk_bf16_fp4, exactly, with their block's scale. The running
// maximum moves only when a score passes it by 2^8, so that most steps have no exchange between
// lanes and no rescaling; what is above 1 costs no precision in fp32 and bf16. Waves meet in LDS.
//
// The work of a batch is the tokens of all its units (sequence, row tile, kv head), in granules of
// 32 W, and a little for each unit's start. As many workgroups as the card holds at once take an equal
// run of it each, found from the lengths on the device: one round, no tail, whatever the lengths are,
// and a graph captured with a batch's limits balances every replay. A unit inside one run is finished
// there; one that crosses runs leaves partial results, at most two a workgroup, for a second launch to
// weigh. Short contexts, and many units of middling ones, take a workgroup a unit and no second launch.
//
// Bounded by HBM where the cache is long and rows are few: 48 sequences of up to 8000 tokens, 32 query
// and 8 kv heads of 128, 208 MB: 46 us, 4.5 TB/s (6.05 is what plain reads reach); one sequence of
// 131072 tokens, 143 MB: 31 us. By the start and the end of a unit where its tokens are few: 8 x 8
// queries of 48 + 16 heads against up to 4000 tokens, 49 MB: 21 us, 8 of them the longest runs' six
// granules, at the read rate. By a step's fixed work (maxima, masks, exchanges, addresses) at heads of 64,
// whose steps read half the bytes: 48 sequences, 32 kv heads, 415 MB: 94 us, 4.4 TB/s. By the launches and
// three dependent reads (length, page, tokens) where it is short: 500 tokens 8 us. The join behind it takes
// 4 to 6.
//
// Every instance keeps 53 to 84 scalars more than there are registers in lanes of vector registers. Three
// spill vector registers to memory, for the most part on the path of NaN blocks: 64 rows at D = 128 (17), 32
// rows at D = 64 (2) and 32 rows at D = 256 in workgroups of 8 waves (39; 4 waves, whose registers suffice,
// took 17.4 us where these took 15.6).
#include <algorithm>

#include "kv4_attn.h"
#include "kv4_attn_shared.h"

namespace kv4 {
namespace {

constexpr int kStep = 32;                   // tokens of a wave's step

// The codes and scales of 16 tokens, as a lane holds them.
template <int D>
struct Raw {
  static constexpr int P = Group<D>::kPlanes;
  typedef typename std::conditional<D >= 128, v4i, v2i>::type Vec;
  Vec k[P], v[P];
  uint32_t ks[P], vs[P];
};

// group: the same in every lane; the lane's share of it is an unsigned 32-bit offset, so the loads
// take a scalar base
template <int D>
__device__ __forceinline__ void load_keys(Raw<D>& w, const uint8_t* group, uint32_t g, uint32_t r) {
  using G = Group<D>;
  typedef typename Raw<D>::Vec Vec;
#pragma unroll
  for (int p = 0; p < G::kPlanes; ++p) {
    w.k[p] = *reinterpret_cast<const Vec*>(
        group + (uint32_t)(G::kKeys + r * (D / 2) + p * 64 + g * sizeof(Vec)));
    // the word that holds the scale (a byte carried to the next step would be masked where it is loaded,
    // with a wait for all that is in flight)
    w.ks[p] = *reinterpret_cast<const uint32_t*>(
        group + (uint32_t)(G::kKeyScales + (D >= 128 ? r * (D / kBlock) + 4 * p : 4 * (r >> 1))));
  }
}
// The bit of its key scales' words that a lane's scale begins at.
template <int D>
__device__ __forceinline__ uint32_t key_scale_bit(uint32_t g, uint32_t r) {
  return D >= 128 ? 8 * g : 16 * (r & 1) + 8 * (g >> 1);
}
template <int D>
__device__ __forceinline__ void load_values(Raw<D>& w, const uint8_t* group, uint32_t g,
                                            uint32_t r) {
  using G = Group<D>;
  typedef typename Raw<D>::Vec Vec;
#pragma unroll
  for (int p = 0; p < G::kPlanes; ++p) {
    w.v[p] = *reinterpret_cast<const Vec*>(
        group + (uint32_t)(G::kValues + ((p * 4 + g) * 16 + r) * sizeof(Vec)));
    w.vs[p] = *reinterpret_cast<const uint32_t*>(
        group + (uint32_t)(G::kValueScales + (D >= 128 ? 4 * p + (r >> 2) : r >> 3) * kGroup + 4 * g));
  }
}

// What a unit costs besides its granules (its queries, the first reads of its pages and tokens, the
// waves' shares, what is written), in granules: 4.5 us against 1.1 to 2.2 a granule. Without it a run of
// several short units was the last to end: 30 sequences of up to 8000 tokens, 4 kv heads of 256: 37.6
// us, 32.4 with it; 8 times 8 queries against up to 4000 tokens: 22.0 and 20.0.
constexpr int kStart = 2;

// Granules of a sequence's units: each of tiles x kv heads units has as many as its visible tokens
// take, one at least (a unit of no tokens writes its zeros, a bad sequence its NaN).
struct Units { int per_unit, units, lo; };
template <int kGranule>
__device__ __forceinline__ Units units_of(const AttnArgs& a, const Sequence& s, int tile_rows) {
  if (s.bad) return {1, a.Hkv, 0};
  const int R = s.n * a.group;
  if (R == 0 || (a.few_rows && R > a.few_rows)) return {1, 0, 0};
  const Span x = query_span(a, s, 0, s.n - 1);
  return {x.hi > x.lo ? ceil_div(x.hi - x.lo, kGranule) : 1, ceil_div(R, tile_rows) * a.Hkv, x.lo};
}

// A run of the batch's work, which is for each unit `start` and its granules: the run's first sequence,
// where in that sequence's work it begins, how much it is, and the runs' size. start is kStart, or 0
// where every unit is a whole number of runs and none begins inside one. Every wave finds its run by
// itself, 64 sequences at a time: no exchange between waves.
struct Run { Sequence s; int b, start; uint32_t off, left, share; };
template <int kGranule>
__device__ __forceinline__ Run find_run(const AttnArgs& a, int tile_rows, int lane) {
  Run run = {{0, 0, 0, false}, 0, 0, 0, 0, 0};
  Sequence s = {0, 0, 0, false};
  Units x = {1, 0, 0};
  auto look = [&](int i) {
    s = {0, 0, 0, false}, x = {1, 0, 0};
    if (i >= a.batch) return;
    s = sequence(a, i);
    x = units_of<kGranule>(a, s, tile_rows);
  };
  auto sum = [](uint32_t n) { return (uint32_t)__builtin_amdgcn_readlane(wave_scan(n), 63); };
  uint32_t granules = 0, units = 0;
  for (int i0 = (a.batch - 1) & ~63; i0 >= 0; i0 -= 64) {
    look(i0 + lane);
    granules += sum((uint32_t)x.per_unit * (uint32_t)x.units), units += sum(x.units);
  }
  run.share = a.by_runs(granules + a.runs - 1);
  bool crosses = false;
  for (int i0 = (a.batch - 1) & ~63; i0 >= 0 && !crosses; i0 -= 64) {
    if (a.batch > 64) look(i0 + lane);
    crosses = __ballot(x.units && run.share && x.per_unit % run.share) != 0;
  }
  if (crosses) run.start = kStart, run.share = a.by_runs(granules + kStart * units + a.runs - 1);
  const uint32_t total = granules + run.start * units, at = run.share * blockIdx.x;
  if (at >= total) return run;           // no work left for this workgroup
  run.left = min(run.share, total - at);
  uint32_t before = 0;
  for (int i0 = 0; i0 < a.batch; i0 += 64) {
    if (a.batch > 64) look(i0 + lane);
    const uint32_t w = (uint32_t)(x.per_unit + run.start) * (uint32_t)x.units, upto = wave_scan(w);
    const uint32_t lo = before + upto - w;
    const uint64_t here = __ballot(at >= lo && at - lo < w);
    if (here) {
      const int k = __builtin_ctzll(here);
      run.b = i0 + k;
      run.off = at - __builtin_amdgcn_readlane(lo, k);
      run.s.len = __builtin_amdgcn_readlane(s.len, k);
      run.s.q0 = __builtin_amdgcn_readlane(s.q0, k);
      run.s.n = __builtin_amdgcn_readlane(s.n, k);
      run.s.bad = __builtin_amdgcn_readlane(s.bad, k);
      return run;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  run.left = 0;
  return run;
}

template <int D, int RF, int W>
struct Shared {
  v4i q[RF * (D / 32)][64];
  float stat[2][W][RF * 16];
  float merge[W][16][D + 4];
};

template <int D, int RF, int W>
__global__ __launch_bounds__(64 * W, attn_waves(D, RF)) void attn_rows(AttnArgs a) {
  using G = Group<D>;
  constexpr int P = G::kPlanes, M = G::kRun, KS = D / 32;   // planes, channels of a run, K steps
  constexpr int kGranule = kStep * W, kTile = 16 * RF;
  __shared__ Shared<D, RF, W> sh;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group_heads = a.group;

  Run run = {{0, 0, 0, false}, 0, 0, 0, 0, 0};
  if (a.tiles) {
    // short contexts: one unit, workgroups [batch][tiles][kv heads]
    const uint32_t per = a.tiles * a.Hkv;
    run.b = blockIdx.x / per;
    run.s = sequence_uniform(a, run.b);
    const Units x = units_of<kGranule>(a, run.s, kTile);
    const uint32_t u = blockIdx.x % per;
    if (u >= (uint32_t)x.units) return;
    run.off = u * x.per_unit, run.left = x.per_unit, run.share = 0;
  } else {
    run = find_run<kGranule>(a, kTile, lane);
    if (tid == 0 && !a.by_unit) meta(a, kTile, D, blockIdx.x)[0] = 0;
    if (!run.left) return;
  }

  const float c = a.scale * 1.44269504088896340736f;
  const float slack = 8.0f / c;
  const int start = run.start;
  int unit = 0, at = 0;       // the unit of the sequence and the place in its work that the run stands at
  {
    const int work = units_of<kGranule>(a, run.s, kTile).per_unit + start;
    if (run.off) {
      unit = __builtin_amdgcn_readfirstlane(run.off / (uint32_t)work);
      at = run.off - unit * work;
    }
  }
  while (true) {
    const Sequence s = run.s;
    const int b = run.b;
    const Units un = units_of<kGranule>(a, s, kTile);
    if (unit >= un.units) {                                 // the next sequence
      if (++run.b >= a.batch) return;
      unit = 0;
      run.s = sequence_uniform(a, run.b);
      continue;
    }
    const int rest = un.per_unit + start - at, part = min((uint32_t)rest, run.left), this_unit = unit;
    const int first_granule = max(at - start, 0), take = max(at + part - start, 0) - first_granule;
    const int tile = a.by_heads(unit), h = unit - tile * a.Hkv;
    const bool whole = take == un.per_unit;
    run.left -= part, at += part;
    if (part == rest) ++unit, at = 0;
    if (take == 0) {          // the run ends within a unit's start: the next one begins it
      if (!run.left) return;
      continue;
    }
    if (s.bad) {
      nan_rows<D>(a, s, h * group_heads, group_heads);
      if (!run.left) return;
      continue;
    }
    const int R = s.n * group_heads, r0 = tile * kTile;
    const Span span = query_span(a, s, a.by_group(r0), a.by_group(min(r0 + kTile, R) - 1));
    const int t0 = un.lo + first_granule * kGranule;
    const int t1 = min(span.hi, t0 + take * kGranule);

    // the rows' query operands, asked for here and put into LDS for all waves behind the first loads
    // of the cache; the tokens that this lane's rows see
    constexpr int kOps = ceil_div(RF * KS, W);
    v4i ops[kOps];
#pragma unroll
    for (int j = 0; j < kOps; ++j) {
      const int i = wave + j * W, k = i % KS;
      const int row = min(r0 + min(i / KS, RF - 1) * 16 + r, R - 1), qi = a.by_group(row);
      const uint16_t* src = a.q + (size_t)(s.q0 + qi) * a.q_ts +
                            (size_t)(h * group_heads + row - qi * group_heads) * a.q_hs;
      ops[j] = *reinterpret_cast<const v4i*>(
          src + (D >= 128 ? 128 * (k >> 2) + 32 * g + 8 * (k & 3) : 16 * g + 8 * k));
    }
    int hi[RF], lo[RF];
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      const int place = s.len - s.n + a.by_group(min(r0 + f * 16 + r, R - 1));
      hi[f] = a.causal ? min(place + 1, s.len) : s.len;
      lo[f] = first_seen(a, place);
    }

    // The page of a step's 16 tokens: its number is read two steps ahead of the tokens' use. Tokens
    // from t1 on read the last page that holds some before it.
    const int* table = a.pages_of + (size_t)b * a.table_stride;
    const uint8_t* head_base = a.cache + (size_t)(h << (a.page_shift - 4)) * G::kBytes;
    const int group_mask = (1 << (a.page_shift - 4)) - 1;
    const int last_page = (t1 - 1) >> a.page_shift;
    auto page_of = [&](int t) { return scalar_load(table + min(t >> a.page_shift, last_page)); };
    auto group_at = [&](int t, int page) {
      return tokens_at(a, head_base, __builtin_amdgcn_readfirstlane(page), (t >> 4) & group_mask, G::kBytes);
    };

    float m[RF], l[RF];                // row maximum (raw scores), this lane's share of the sum
    v4f o[RF][P][M];
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      m[f] = -INFINITY, l[f] = 0.0f;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < M; ++i) o[f][p][i] = v4f{0, 0, 0, 0};
    }

    // A step's codes in registers: the next step's keys are asked for when this one's scores are done,
    // its values when this one's products are (two and three steps ahead measured the same). Past the
    // end the segment's last step is asked for again (cache hits that nothing uses): loads that are
    // always issued let the waits count those in flight instead of draining them.
    Raw<D> w[2];
    const uint32_t ks_bit = key_scale_bit<D>(g, r);
    const int t_last = (t1 - 1 - t0) / kStep * kStep + t0;
    int t = t0 + wave * kStep;
    int na = 0, nb = 0;                // page numbers of the next step to ask for
    Tokens ta = {}, tb = {};           // whose keys are in w
    if (t < t1) {
      ta = group_at(t, page_of(t)), tb = group_at(t + 16, page_of(t + 16));
      load_keys<D>(w[0], ta.group, g, r), load_keys<D>(w[1], tb.group, g, r);
      load_values<D>(w[0], ta.group, g, r), load_values<D>(w[1], tb.group, g, r);
      const int tn = min(t + kGranule, t_last);
      na = page_of(tn), nb = page_of(tn + 16);
    }
#pragma unroll
    for (int j = 0; j < kOps; ++j)
      if (wave + j * W < RF * KS) sh.q[wave + j * W][lane] = ops[j];
    __syncthreads();
    for (; t < t1; t += kGranule) {
      // (A branch: two more values in the products' loop spill registers. Here and below the compiler is
      // told that it is seldom taken: without, 4 sequences of 500 tokens, 5 queries, 24 and 4 heads of 256
      // took 16.9 us in place of 16.0.)
      if (__builtin_expect((ta.nan | tb.nan) != 0, 0)) {
#pragma unroll
        for (int p = 0; p < P; ++p) w[0].ks[p] |= ta.nan, w[1].ks[p] |= tb.nan;
      }
      // scores of 2 x 16 tokens: lane holds tokens 4 g + i of both, row r
      v4f sc[RF][2];
#pragma unroll
      for (int f = 0; f < RF; ++f) sc[f][0] = sc[f][1] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int p = D >= 128 ? k >> 2 : 0;
        const v8bf k0 = expand8(w[0].k[p][D >= 128 ? k & 3 : k], stored_scale((w[0].ks[p] >> ks_bit) & 0xFFu));
        const v8bf k1 = expand8(w[1].k[p][D >= 128 ? k & 3 : k], stored_scale((w[1].ks[p] >> ks_bit) & 0xFFu));
#pragma unroll
        for (int f = 0; f < RF; ++f) {
          const v8bf q = __builtin_bit_cast(v8bf, sh.q[f * KS + k][lane]);
          sc[f][0] = mfma16(k0, q, sc[f][0]);
          sc[f][1] = mfma16(k1, q, sc[f][1]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      const int tn = min(t + kGranule, t_last);
      ta = group_at(tn, na), tb = group_at(tn + 16, nb);
      load_keys<D>(w[0], ta.group, g, r), load_keys<D>(w[1], tb.group, g, r);
      const int tp = min(tn + kGranule, t_last);
      na = page_of(tp), nb = page_of(tp + 16);
      if (t + kStep > span.all_hi || t < span.all_lo) {   // tokens that some row does not see
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int tok = t + 16 * u + 4 * g + i;
              if (tok >= hi[f] || tok < lo[f]) sc[f][u][i] = -INFINITY;
            }
      }
      v8bf pr[RF];
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        float mx = fmaxf(fmaxf(fmaxf(sc[f][0][0], sc[f][0][1]), fmaxf(sc[f][0][2], sc[f][0][3])),
                         fmaxf(fmaxf(sc[f][1][0], sc[f][1][1]), fmaxf(sc[f][1][2], sc[f][1][3])));
        if (__ballot(mx > m[f] + slack)) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float mn = fmaxf(m[f], mx);
          const float alpha = mn == m[f] ? 1.0f : exp2_raw((m[f] - mn) * c);
          m[f] = mn;
          l[f] *= alpha;
#pragma unroll
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < M; ++i) o[f][p][i] *= alpha;
        }
        const float sub = m[f] == -INFINITY ? 0.0f : m[f] * c;
        float e[8];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) e[4 * u + i] = exp2_raw(fmaf(sc[f][u][i], c, -sub));
        l[f] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        pr[f] = pack8bf(e);
      }
      // A NaN block of a token that a row does not see (a later query's, or nobody's behind the last
      // token): its product with a weight of zero would reach the row. Such blocks are taken out of
      // the values, and the rows that do see them are marked through a product of its own.
      uint32_t nan = 0;
#pragma unroll
      for (int p = 0; p < P; ++p) nan |= nan_scales(w[0].vs[p]) | nan_scales(w[1].vs[p]);
      if (__builtin_expect(__ballot(nan != 0) != 0, 0)) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float is[8];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t hit = nan_scales(w[u].vs[p]);
#pragma unroll
            for (int i = 0; i < 4; ++i) is[4 * u + i] = hit >> (8 * i) & 0xFFu ? 1.0f : 0.0f;
            w[u].vs[p] &= ~((hit >> 7) * 0xFFu);
          }
          const v8bf mark = pack8bf(is);
#pragma unroll
          for (int f = 0; f < RF; ++f) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int tok = t + 16 * u + 4 * g + i;
                is[4 * u + i] = tok < hi[f] && tok >= lo[f] ? 1.0f : 0.0f;
              }
            const v4f hit = mfma16(mark, pack8bf(is), v4f{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (hit[x] > 0.0f) o[f][p][i][x] = __uint_as_float(0x7FC00000u);
          }
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
        each_value_pair<D>(w[0].v[p], w[0].vs[p], w[1].v[p], w[1].vs[p],
                           [&](auto pair, v8bf even, v8bf odd) {
                             constexpr int i = 2 * decltype(pair)::value;
#pragma unroll
                             for (int f = 0; f < RF; ++f) {
                               o[f][p][i] = mfma16(even, pr[f], o[f][p][i]);
                               o[f][p][i + 1] = mfma16(odd, pr[f], o[f][p][i + 1]);
                             }
                             __builtin_amdgcn_sched_barrier(0);
                           });
      load_values<D>(w[0], ta.group, g, r), load_values<D>(w[1], tb.group, g, r);
    }

    // ---- the waves' shares -----------------------------------------------------------------------
    {
    // (tid pinned here, or the addresses below are kept in registers through the steps)
    const int tid = pinned(threadIdx.x), lane = tid & 63, g = lane >> 4, r = lane & 15;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      l[f] += __shfl_xor(l[f], 16);
      l[f] += __shfl_xor(l[f], 32);
      if (g == 0) sh.stat[0][wave][f * 16 + r] = m[f], sh.stat[1][wave][f * 16 + r] = l[f];
    }
    __syncthreads();
    const int which = first_granule > 0 ? 0 : 1;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, sh.stat[0][w][f * 16 + r]);
      const float mine = m[f] == top ? 1.0f : exp2_raw((m[f] - top) * c);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // channels of the plane: M * (4 g + x) + i
#pragma unroll
          for (int i = 0; i < M; i += 4) {
            const v4f y = {o[f][p][i][x] * mine, o[f][p][i + 1][x] * mine,
                           o[f][p][i + 2][x] * mine, o[f][p][i + 3][x] * mine};
            *reinterpret_cast<v4f*>(&sh.merge[wave][r][p * 128 + M * (4 * g + x) + i]) = y;
          }
        }
      __syncthreads();
      // 16 rows x D: each thread C channels of one row
      constexpr int kThreads = 64 * W / 16, C = D / kThreads < 4 ? 4 : D / kThreads;
      const int row = tid / kThreads, ch = tid % kThreads * C;
      const int tr = r0 + f * 16 + row;
      if (ch < D && tr < R) {
        float tm = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) tm = fmaxf(tm, sh.stat[0][w][f * 16 + row]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float wm = sh.stat[0][w][f * 16 + row];
          sum += sh.stat[1][w][f * 16 + row] * (wm == tm ? 1.0f : exp2_raw((wm - tm) * c));
        }
        float y[C];
#pragma unroll
        for (int i = 0; i < C; i += 4) {
          v4f acc = {0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < W; ++w)
            acc += *reinterpret_cast<const v4f*>(&sh.merge[w][row][ch + i]);
          y[i] = acc[0], y[i + 1] = acc[1], y[i + 2] = acc[2], y[i + 3] = acc[3];
        }
        if (whole) {
          if (!sees_any(a, s.len, s.len - s.n + a.by_group(tr))) sum = INFINITY;
          store_row<C>(out_row(a, D, s.q0, h, tr) + ch, y, sum);
        } else {
          store_part<C>(a, kTile, D, 2 * blockIdx.x + which, f * 16 + row, ch, y, tm * c, sum);
        }
      }
      __syncthreads();
    }
    }
    if (a.runs && first_granule == 0 && tid == 0 && (a.by_unit || !whole)) {
      // what attn_join is told of a unit: how many workgroups after this one finish it
      int* mt = meta(a, kTile, D, a.by_unit ? b * a.units + this_unit : blockIdx.x);
      // (no more than there are: starts that go back can make more work than 32 bits count)
      mt[0] = min((int)((rest - part + run.share - 1) / run.share), a.runs - 1 - (int)blockIdx.x);
      mt[1] = b, mt[2] = this_unit, mt[3] = blockIdx.x;
    }
    if (!run.left) return;
  }
}

// A unit that crosses runs: the partial results of workgroup i (its last) and of the n after it (their
// first), weighed. D / 4 threads read a partial result of a row, S such teams share a row's. What a
// unit's first workgroup has written is found by the unit, or by that workgroup where those are
// fewer. The rows of 8 partial results a thread are read without waiting for the maxima that weigh
// them.
template <int D, int S>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a, int tile_rows, int entries, int rows) {
  constexpr int kLanes = D / 4, kTeams = 256 / kLanes, kRows = kTeams / S, kAhead = 8;
  __shared__ v4f side[S > 1 ? kTeams : 1][kLanes];
  __shared__ float sums[kTeams];
  const int tid = threadIdx.x, lane = tid % kLanes, team = tid / kLanes, mine = team % S;
  const int entry = blockIdx.x % entries, row = blockIdx.x / entries * kRows + team / S;
  const int* mt = meta(a, tile_rows, D, entry);
  int n = mt[0], b = mt[1], unit = mt[2];
  const int i0 = mt[3];
  if (a.by_unit) {
    // a unit that the batch does not have was not written
    b = entry / a.units, unit = entry % a.units;
    const Sequence s = sequence_uniform(a, b);
    const int R = s.n * a.group;
    if (s.bad || a.by_heads(unit) * tile_rows >= R || (a.few_rows && R > a.few_rows)) return;
  }
  if (!n) return;
  const int tile = a.by_heads(unit), h = unit - tile * a.Hkv;
  const int len = scalar_load(a.lens + b), q0 = scalar_load(a.starts + b);
  const int queries = scalar_load(a.starts + b + 1) - q0, R = queries * a.group;
  const int tr = tile * tile_rows + row;
  const int last = row < rows && tr < R ? n : -1;        // no partial results of a row beyond
  // partial 0 is the last of workgroup i0, partial k > 0 the first of workgroup i0 + k
  // (those of a unit that attn_tiles did in parts lie one after the other)
  auto slot = [&](int k) { return a.by_parts ? i0 + k : 2 * (i0 + k) + (k == 0 ? 1 : 0); };
  v4f part[kAhead];
  float st[kAhead][2];
  auto read = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = k0 + j * S;
      if (k > last) break;
      part[j] = *reinterpret_cast<const v4f*>(part_row(a, tile_rows, D, slot(k), row) + 4 * lane);
      const float* p = part_stat(a, tile_rows, D, slot(k), row);
      st[j][0] = p[0], st[j][1] = p[1];
    }
  };
  read(mine);
  float top = -INFINITY;
  for (int k = lane; k <= last; k += kLanes)
    top = fmaxf(top, part_stat(a, tile_rows, D, slot(k), row)[0]);
#pragma unroll
  for (int x = 1; x < kLanes; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  float sum = 0.0f;
  v4f y = {0, 0, 0, 0};
  for (int k0 = mine; k0 <= last;) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (k0 + j * S > last) break;
      const float w = st[j][0] == top ? 1.0f : exp2_raw(st[j][0] - top);
      sum += w * st[j][1];
      y += w * part[j];
    }
    k0 += kAhead * S;
    read(k0);
  }
  if constexpr (S > 1) {
    side[team][lane] = y;
    if (lane == 0) sums[team] = sum;
    __syncthreads();
    if (mine) return;
#pragma unroll
    for (int k = 1; k < S; ++k) y += side[team + k][lane], sum += sums[team + k];
  }
  if (last < 0) return;
  const float out[4] = {y[0], y[1], y[2], y[3]};
  if (!sees_any(a, len, len - queries + a.by_group(tr))) sum = INFINITY;
  store_row<4>(out_row(a, D, q0, h, tr) + 4 * lane, out, sum);
}

// rows: of a sequence at most
template <int D>
hipError_t join(const AttnArgs& a, int tile_rows, int entries, int rows, hipStream_t stream) {
  if (rows > tile_rows) rows = tile_rows;
  // A row to a workgroup where the rows are few: many workgroups' partial results each. A row to a
  // team where they are many (of few partial results each).
  constexpr int kTeams = 1024 / D;
  if ((long)entries * rows <= 2048)
    attn_join<D, kTeams><<<entries * rows, 256, 0, stream>>>(a, tile_rows, entries, rows);
  else
    attn_join<D, 1><<<entries * ceil_div(rows, kTeams), 256, 0, stream>>>(a, tile_rows, entries, rows);
  return hipGetLastError();
}

template <int D, int RF>
hipError_t launch(AttnArgs a, hipStream_t stream) {
  constexpr int W = kRunWaves;
  const int rows = a.few_rows ? a.few_rows : std::max(a.max_q, 1) * a.group;   // of a sequence at most
  a.by_group = divisor(a.group), a.by_heads = divisor(a.Hkv), a.by_runs = divisor(a.runs ? a.runs : 1);
  if (!a.runs) {
    a.tiles = ceil_div(rows, 16 * RF);
    constexpr int WW = attn_whole_waves(RF);
    attn_rows<D, RF, WW><<<a.batch * a.tiles * a.Hkv, 64 * WW, 0, stream>>>(a);
    return hipGetLastError();
  }
  a.tiles = 0;
  a.units = ceil_div(rows, 16 * RF) * a.Hkv;
  a.by_unit = (long)a.batch * a.units <= a.runs;
  attn_rows<D, RF, W><<<a.runs, 64 * W, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return join<D>(a, 16 * RF, a.by_unit ? a.batch * a.units : a.runs, rows, stream);
}

template <int D>
hipError_t launch_d(const AttnArgs& a, hipStream_t stream) {
  switch (a.fragments) {
    case 1: return launch<D, 1>(a, stream);
    case 2: return launch<D, 2>(a, stream);
    default:
      if constexpr (D <= 128) return launch<D, 4>(a, stream);
      return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_attn_join(const AttnArgs& a, int d, int tile_rows, int entries, hipStream_t stream) {
  return d == 64 ? join<64>(a, tile_rows, entries, tile_rows, stream)
                 : d == 128 ? join<128>(a, tile_rows, entries, tile_rows, stream)
                            : join<256>(a, tile_rows, entries, tile_rows, stream);
}

// Partial results of attn_tiles at most: two for each CU, 68 MB.
constexpr int kMostEntries = 2 * kCUs;

AttnPlan attn_plan(int total, int batch, int max_q, int max_len, int Hq, int Hkv, int d, int window) {
  const int group = Hq / Hkv;
  const long rows = (long)max_q * group;
  AttnPlan p = {};
  // Row fragments: the fewest of 1, 2, 4 that hold a sequence's rows, 4 (2 at D = 256, whose
  // accumulators are twice as wide) beyond.
  auto fragments = [d](long n) { return n <= 16 ? 1 : n <= 32 || d == 256 ? 2 : 4; };
  // tokens that a row tile can see
  long span = max_len;
  if (window > 0 && (long)window + max_q + 31 < span) span = (long)window + max_q + 31;
  long few = rows;
  // attn_tiles or attn_rows: a workgroup of attn_tiles does what four row tiles (of 64 rows, 32 at
  // D = 256) of attn_rows do, in the time of 2.6 of them; but it has a CU to itself, so that few of
  // them are cut into parts, each with a start, an end and partial results of its own. Against 4096
  // cached tokens, attn_tiles and attn_rows with attn_join in us a call:
  //   d = 128, 32 query and 8 kv heads        d = 256, 24 and 4                 d = 64, 64 and 8
  //   1 x 128 queries    64 tiles  28  32     1 x 100  76 tiles  39  42         1 x 64    64 tiles  20  23
  //   1 x 256           128        38  40     1 x 512 384        96 124         1 x 512  512        53  61
  //   1 x 512           256        49  57     4 x 256 768       161 229
  //   1 x 1024          512        79  83                                       and 32 and 32 heads of 64:
  //   1 x 4096         2048       137 273                                       1 x 600  320        51  52
  //   16 x 33 (132 rows) 384       74  80
  // Decoding sequences beside a chunk in attn_rows are read with the chunk's 64 rows: with 100 MB of cache
  // and more that costs more than the two launches of attn_rows beside attn_tiles do: one chunk and 47
  // sequences of 4000 tokens, d = 128, 64 queries: 73 and 78, 256: 83 and 83; 100 queries and 7
  // sequences of 3000: 42 and 35.
  const long rows_tile = d == 256 ? 32 : 64;
  // all sequences have max_q queries
  const bool even = total == (long)batch * max_q;
  // Row tiles of the batch at most: a sequence (or bad one) has one that is not full.
  auto tiles_of_batch = [&](long tile) {
    const long each = batch * ((rows + tile - 1) / tile), all = (long)total * group / tile + batch;
    return even || each < all ? each : all;
  };
  if (rows > 2 * rows_tile && ((long)total * Hq >= 200 * rows_tile || (!even && (long)batch * span * Hkv * d >= 100000000))) {
    p.tiles = true;
    const long tile_rows = attn_tile_rows(d), units = tiles_of_batch(tile_rows) * Hkv;
    p.units = (int)units;
    p.span = span;
    // The last round of row tiles is done in parts: into how many is known here where the batch is even.
    if (even) {
      const int rest = (int)(units % kCUs), parts = attn_parts(rest, span, kMostEntries);
      p.entries = parts > 1 ? rest * parts : 0;
    } else {
      p.entries = (int)(units * 16 < kMostEntries ? units * 16 : kMostEntries);
    }
    p.threads = (units + p.entries) * attn_tile_rows(d) * 2;     // 64 for each 32 rows
    if (p.entries)
      p.tiles_workspace = p.workspace =
          (size_t)(p.entries + 1) / 2 * 2 * tile_rows * (d + 2) * sizeof(float) + kCUs * 16;
    // Sequences of fewer queries beside: those of one query are attn_rows', and those of as many as the
    // others have beside the longest on average, where they fit (40 sequences of 8 queries and 3000 tokens
    // beside a chunk of 300, d = 128: 81 us, 150 in attn_tiles).
    if (even) return p;
    const long others = batch > 1 ? ((long)total - max_q + batch - 2) / (batch - 1) * group : 0;
    const long want = others <= rows_tile && others > group ? others : group;
    const int fit = want <= 16 ? 16 : want <= 32 || d == 256 ? 32 : 64;
    if (group > fit) return p;
    few = p.few_rows = fit;
  }
  p.rows = true;
  p.fragments = fragments(few);
  const int tile = 16 * p.fragments;
  const long most_units = (long)batch * Hkv * ((few + tile - 1) / tile);
  const long units = p.few_rows ? most_units : tiles_of_batch(tile) * Hkv;
  // A workgroup a unit, and no second launch, where its waves have few steps to go, or the units are many
  // and of like length enough. Equal lengths L, such workgroups and runs with the join, us a call (d = 128,
  // 32 query and 8 kv heads unless said):
  //   L = 1000, 1 sequence   9.7   9.9    L = 2000, 1    13.8  10.2    L = 3000, 32     20.5  25.5
  //                    16   10.0  14.3              4    14.1  11.6             100     66.2  68.1
  //                    64   16.5  22.3             16    14.3  16.1    L = 6000, 16     30.2  26.9
  //   8 queries (32 rows)                         200    85.5  96.6    200 .. 6000, 48  43.1  36.8
  //   L = 800, 8 sequences  12.4  17.6    8 x 3 rows, 16 kv heads, L = 2000: 14.0  15.9, L = 3000: 18.4  17.9
  const long waves_step = kStep * attn_whole_waves(p.fragments), steps = (span + waves_step - 1) / waves_step;
  // (not where most of those workgroups would have nothing to do)
  if (most_units <= 2 * units && (steps <= 4 || (span <= (p.fragments == 1 ? 4096 : 2048) && units >= 16 * steps))) {
    p.threads = std::max(p.threads, most_units * 64 * attn_whole_waves(p.fragments));
    return p;
  }
  // as many workgroups as the card's 256 CUs hold at once, or a granule each
  const long granules = (span + kStep * kRunWaves - 1) / (kStep * kRunWaves);
  const long most = 256L * 4 * attn_waves(d, p.fragments) / kRunWaves;
  p.runs = (int)(units * granules < most ? units * granules : most);
  // (where attn_join looks at every unit there may be, all of them count)
  p.work = (most_units <= p.runs ? most_units : units) * (granules + kStart);
  p.workspace += (size_t)p.runs * ((size_t)2 * tile * (d + 2) * sizeof(float) + 16);
  return p;
}

hipError_t launch_attn_rows(const AttnArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch_d<64>(a, stream)
                 : d == 128 ? launch_d<128>(a, stream) : launch_d<256>(a, stream);
}

}  // namespace kv4
