// Attention over the 4-bit paged cache for gfx950, few query rows: decode, speculative verify.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c s_j - m),  s_j = q . k_j,  c = scale * log2(e)
//
// The rows of one kv head are its sequence's queries times the query heads that share it; a
// workgroup has 16 * RF of them and one chunk of the cached tokens, its four waves 32 tokens at a
// time in turn. Keys and values are read once, straight into registers in matrix-operand order:
//   S^T = K . Q^T   (16 tokens x 16 rows): lane (g = l / 16, r = l % 16) holds token r, one block of
//                   32 channels per instruction group; its 16 bytes of codes and one scale.
//   O^T = V^T . P^T (16 channels x 16 rows over 32 tokens): the scores' registers are already the
//                   P^T operand (tokens 4 g + i of both groups of 16), and the value layout gives a
//                   lane the same 8 tokens of the 8 channels of run r.
// Codes become bf16 by v_cvt_scalef32_pk_bf16_fp4, exactly, with their block's scale. The running
// maximum moves only when a score passes it by 2^8, so that most steps have no exchange between
// lanes and no rescaling; what is above 1 costs no precision in fp32 and bf16. Waves meet in LDS,
// chunks in a second launch that weighs the partial results.
//
// Bounded by HBM where the cache is long; by the launches and three dependent reads (length, page,
// tokens) where it is short.
#include "kv4_attn.h"
#include "kv4_attn_shared.h"

namespace kv4 {
namespace {

constexpr int kWaves = 4;
constexpr int kStep = 32;                   // tokens of a wave's step

// The codes and scales of 16 tokens, as a lane holds them.
template <int D>
struct Raw {
  static constexpr int P = Group<D>::kPlanes;
  typedef typename std::conditional<D >= 128, v4i, v2i>::type Vec;
  Vec k[P], v[P];
  uint32_t ks[P], vs[P];
};

template <int D>
__device__ __forceinline__ void load_group(Raw<D>& w, const uint8_t* group, int g, int r) {
  using G = Group<D>;
  typedef typename Raw<D>::Vec Vec;
  constexpr int B = sizeof(Vec);
#pragma unroll
  for (int p = 0; p < G::kPlanes; ++p) {
    w.k[p] = *reinterpret_cast<const Vec*>(group + G::kKeys + r * (D / 2) + p * 64 + g * B);
    w.v[p] = *reinterpret_cast<const Vec*>(group + G::kValues + ((p * 4 + g) * 16 + r) * B);
    w.ks[p] = group[G::kKeyScales + r * (D / kBlock) + (D >= 128 ? 4 * p + g : g >> 1)];
    w.vs[p] = *reinterpret_cast<const uint32_t*>(
        group + G::kValueScales + (D >= 128 ? 4 * p + (r >> 2) : r >> 3) * kGroup + 4 * g);
  }
}

template <int D, int RF>
__global__ __launch_bounds__(256) void attn_rows(AttnArgs a, int tiles) {
  using G = Group<D>;
  constexpr int P = G::kPlanes, M = G::kRun, KS = D / 32;   // planes, channels of a run, K steps
  constexpr int kPad = D + 4;
  __shared__ int pages[kMaxChunk / 16 + 1];
  __shared__ int bad_page;
  __shared__ float stat[2][kWaves][RF * 16];
  __shared__ float merge[kWaves][16][kPad];

  // workgroups: [batch][row tiles][kv heads][splits]
  const int group_heads = a.Hq / a.Hkv;
  const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int h = rest % a.Hkv, tile = rest / a.Hkv % tiles, b = rest / a.Hkv / tiles;
  const Sequence s = sequence(a, b);
  if (s.bad) {
    if (split == 0 && tile == 0) nan_rows<D>(a, s, h * group_heads, group_heads);
    return;
  }
  const int R = s.n * group_heads, r0 = tile * 16 * RF;
  if (r0 >= R) return;
  const Span span = tile_span(a, s, r0, min(r0 + 16 * RF, R) - 1, group_heads);
  const int t0 = span.lo + split * a.chunk;
  const int t1 = min(span.hi, t0 + a.chunk);
  const bool direct = span.hi - span.lo <= a.chunk;     // one chunk: no partial results
  if (t0 >= t1 && !(direct && split == 0)) return;

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, r = lane & 15;
  const int first_page = t0 >> a.page_shift;
  const int npages = t1 > t0 ? ((t1 - 1) >> a.page_shift) - first_page + 1 : 0;
  if (tid == 0) bad_page = 0;
  __syncthreads();
  for (int i = tid; i < npages; i += 256) {
    const int p = a.pages_of[(size_t)b * a.table_stride + first_page + i];
    const bool ok = p >= 0 && p < a.pages;
    pages[i] = ok ? p : 0;
    if (!ok) bad_page = 1;
  }

  // this lane's rows: query operand, and the tokens they see
  v8bf q[RF][KS];
  int hi[RF], lo[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const int row = r0 + f * 16 + r;
    const int qi = min(row, R - 1) / group_heads, head = min(row, R - 1) % group_heads;
    const int place = s.len - s.n + qi;
    hi[f] = a.causal ? min(place + 1, s.len) : s.len;
    lo[f] = a.window > 0 ? place - a.window + 1 : 0;
    const uint16_t* src = a.q + (size_t)(s.q0 + qi) * a.q_ts + (size_t)(h * group_heads + head) * a.q_hs;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      q[f][k] = __builtin_bit_cast(
          v8bf, *reinterpret_cast<const v4i*>(
                    src + (D >= 128 ? 128 * (k >> 2) + 32 * g + 8 * (k & 3) : 16 * g + 8 * k)));
  }
  __syncthreads();

  const uint8_t* head_base = a.cache + (size_t)(h << (a.page_shift - 4)) * G::kBytes;
  const int group_mask = (1 << (a.page_shift - 4)) - 1;
  auto group_at = [&](int t) {
    const int i = min((t >> a.page_shift) - first_page, npages - 1);
    const int p = __builtin_amdgcn_readfirstlane(pages[i]);
    return head_base + (size_t)p * a.page_stride + (size_t)((t >> 4) & group_mask) * G::kBytes;
  };

  const float c = a.scale * 1.44269504088896340736f;
  const float slack = 8.0f / c;
  float m[RF], l[RF];                  // row maximum (raw scores), this lane's share of the sum
  v4f o[RF][P][M];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    m[f] = -INFINITY, l[f] = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < M; ++i) o[f][p][i] = v4f{0, 0, 0, 0};
  }

  Raw<D> cur[2], nxt[2];
  int t = t0 + wave * kStep;
  if (t < t1) {
    load_group<D>(cur[0], group_at(t), g, r);
    load_group<D>(cur[1], group_at(t + 16), g, r);
  }
  for (; t < t1; t += kWaves * kStep) {
    const int tn = t + kWaves * kStep;
    if (tn < t1) {
      load_group<D>(nxt[0], group_at(tn), g, r);
      load_group<D>(nxt[1], group_at(tn + 16), g, r);
    }
    // scores of 2 x 16 tokens: lane holds tokens 4 g + i of both, row r
    v4f sc[RF][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int f = 0; f < RF; ++f) sc[f][u] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int p = D >= 128 ? k >> 2 : 0;
        const v8bf kf = expand8(cur[u].k[p][D >= 128 ? k & 3 : k], scale_of(cur[u].ks[p]));
#pragma unroll
        for (int f = 0; f < RF; ++f)
          sc[f][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[f][k], sc[f][u], 0, 0, 0);
      }
    }
    // tokens that some row of the tile does not see
    const bool edge = t + kStep > span.all_hi || t < span.all_lo;
    if (edge) {
#pragma unroll
      for (int f = 0; f < RF; ++f)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = t + 16 * u + 4 * g + i;
            if (tok >= hi[f] || tok < lo[f]) sc[f][u][i] = -INFINITY;
          }
      // what lies behind the last token that any row sees is not the sequence's: its values are
      // zeroed, whatever they hold
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + 16 * u + 4 * g + i >= t1)
#pragma unroll
            for (int p = 0; p < P; ++p) cur[u].vs[p] &= ~(0xFFu << (8 * i));
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
    if (edge) {
      // A NaN block of a token that some rows see and others do not: its product with a weight of
      // zero would reach the rows that do not. It is taken out of the values, and the rows that
      // see it are marked through a product of its own.
      bool any = false;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int p = 0; p < P; ++p) any |= has_nan_scale(cur[u].vs[p]);
      if (__ballot(any)) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float isnan[8];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t e = (cur[u].vs[p] >> (8 * i)) & 0xFFu;
              isnan[4 * u + i] = e == 0xFFu ? 1.0f : 0.0f;
              if (e == 0xFFu) cur[u].vs[p] &= ~(0xFFu << (8 * i));
            }
          const v8bf mark = pack8bf(isnan);
#pragma unroll
          for (int f = 0; f < RF; ++f) {
            float sees[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int tok = t + 16 * u + 4 * g + i;
                sees[4 * u + i] = tok < hi[f] && tok >= lo[f] ? 1.0f : 0.0f;
              }
            const v4f hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mark, pack8bf(sees),
                                                                    v4f{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (hit[x] > 0.0f) o[f][p][i][x] = __uint_as_float(0x7FC00000u);
          }
        }
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      v8bf vf[M];
      value_operands<D>(vf, cur[0].v[p], cur[0].vs[p], cur[1].v[p], cur[1].vs[p]);
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int f = 0; f < RF; ++f)
          o[f][p][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i], pr[f], o[f][p][i], 0, 0, 0);
    }
    cur[0] = nxt[0];
    cur[1] = nxt[1];
  }

  // ---- the waves' shares -------------------------------------------------------------------------
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    l[f] += __shfl_xor(l[f], 16);
    l[f] += __shfl_xor(l[f], 32);
    if (g == 0) stat[0][wave][f * 16 + r] = m[f], stat[1][wave][f * 16 + r] = l[f];
  }
  __syncthreads();
  const bool poison = bad_page != 0;
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stat[0][w][f * 16 + r]);
    const float mine = m[f] == top ? 1.0f : exp2_raw((m[f] - top) * c);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        // channels of the plane: M * (4 g + x) + i
#pragma unroll
        for (int i = 0; i < M; i += 4) {
          const v4f y = {o[f][p][i][x] * mine, o[f][p][i + 1][x] * mine, o[f][p][i + 2][x] * mine,
                         o[f][p][i + 3][x] * mine};
          *reinterpret_cast<v4f*>(&merge[wave][r][p * 128 + M * (4 * g + x) + i]) = y;
        }
      }
    __syncthreads();
    // 16 rows x D: each thread D / 16 channels of one row
    constexpr int C = D / 16;
    const int row = tid >> 4, ch = (tid & 15) * C;
    const int tr = r0 + f * 16 + row;
    float tm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) tm = fmaxf(tm, stat[0][w][f * 16 + row]);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float wm = stat[0][w][f * 16 + row];
      sum += stat[1][w][f * 16 + row] * (wm == tm ? 1.0f : exp2_raw((wm - tm) * c));
    }
    if (poison) sum = __uint_as_float(0x7FC00000u);
    float y[C];
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      v4f acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        acc += *reinterpret_cast<const v4f*>(&merge[w][row][ch + i]);
      y[i] = acc[0], y[i + 1] = acc[1], y[i + 2] = acc[2], y[i + 3] = acc[3];
    }
    if (tr < R) {
      if (direct)
        store_row<C>(a.out + ((size_t)(s.q0 + tr / group_heads) * a.Hq + h * group_heads +
                              tr % group_heads) * D + ch, y, sum);
      else
        store_part<D, C>(a, b, h, split, tr, ch, y, tm * c, sum);
    }
    __syncthreads();
  }
}

// Partial results of a row's chunks, weighed: one wave a row.
template <int D>
__global__ __launch_bounds__(256) void attn_join(AttnArgs a, int tile_rows, int rows) {
  constexpr int C = D / 64;
  const int lane = threadIdx.x & 63, fours = ceil_div(rows, 4);
  const int rest = blockIdx.x / fours, h = rest % a.Hkv, b = rest / a.Hkv;
  const int row = blockIdx.x % fours * 4 + (int)(threadIdx.x >> 6);
  const int group_heads = a.Hq / a.Hkv;
  const Sequence s = sequence(a, b);
  const int R = s.n * group_heads;
  if (s.bad || row >= rows || row >= R) return;
  const int r0 = row / tile_rows * tile_rows;
  const Span span = tile_span(a, s, r0, min(r0 + tile_rows, R) - 1, group_heads);
  const int n = span.hi - span.lo <= a.chunk ? 1 : ceil_div(span.hi - span.lo, a.chunk);
  if (n <= 1) return;                         // already written
  float top = -INFINITY;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, part_stat(a, D, b, h, i, row)[0]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  float sum = 0.0f, y[C];
#pragma unroll
  for (int i = 0; i < C; ++i) y[i] = 0.0f;
  for (int i = 0; i < n; ++i) {
    const float* st = part_stat(a, D, b, h, i, row);
    const float w = st[0] == top ? 1.0f : exp2_raw(st[0] - top);
    const float* o = part_row(a, D, b, h, i, row) + lane * C;
    sum += w * st[1];
#pragma unroll
    for (int k = 0; k < C; ++k) y[k] += w * o[k];
  }
  store_row<C>(a.out + ((size_t)(s.q0 + row / group_heads) * a.Hq + h * group_heads +
                        row % group_heads) * D + lane * C, y, sum);
}

template <int D, int RF>
hipError_t launch(const AttnArgs& a, hipStream_t stream) {
  const int rows = a.max_q * (a.Hq / a.Hkv);
  const int tiles = ceil_div(rows, 16 * RF);
  attn_rows<D, RF><<<a.batch * tiles * a.Hkv * a.splits, 256, 0, stream>>>(a, tiles);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) return e;
  attn_join<D><<<a.batch * a.Hkv * ceil_div(rows, 4), 256, 0, stream>>>(a, 16 * RF, rows);
  return hipGetLastError();
}

template <int D>
hipError_t launch_d(const AttnArgs& a, hipStream_t stream) {
  switch (attn_row_fragments(a.max_q, a.Hq, a.Hkv, D)) {
    case 1: return launch<D, 1>(a, stream);
    case 2: return launch<D, 2>(a, stream);
    default:
      if constexpr (D <= 128) return launch<D, 4>(a, stream);
      return launch<D, 2>(a, stream);
  }
}

}  // namespace

// Row fragments of a workgroup: the fewest of 1, 2, 4 that hold a sequence's rows, 4 (2 at D = 256,
// whose accumulators are twice as wide) beyond.
int attn_row_fragments(int max_q, int Hq, int Hkv, int d) {
  const long rows = (long)max_q * (Hq / Hkv);
  return rows <= 16 ? 1 : rows <= 32 || d == 256 ? 2 : 4;
}

AttnPlan attn_plan(int batch, int max_q, int max_len, int Hq, int Hkv, int d, int window) {
  const long rows = (long)max_q * (Hq / Hkv);
  const int tile = 16 * attn_row_fragments(max_q, Hq, Hkv, d);
  const long units = (long)batch * Hkv * ((rows + tile - 1) / tile);
  // tokens that a tile can see
  long span = max_len;
  if (window > 0 && (long)window + max_q + 31 < span) span = (long)window + max_q + 31;
  const int grain = kWaves * kStep;
  long chunk = (span * units / 2048 + grain - 1) / grain * grain;
  chunk = chunk < grain ? grain : chunk > kMaxChunk ? kMaxChunk : chunk;
  AttnPlan p;
  p.chunk = (int)chunk;
  p.splits = (int)((span + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  p.workspace = p.splits == 1 ? 0 : (size_t)batch * Hkv * p.splits * rows * (d + 2) * sizeof(float);
  return p;
}

hipError_t launch_attn(const AttnArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch_d<64>(a, stream)
                 : d == 128 ? launch_d<128>(a, stream) : launch_d<256>(a, stream);
}

}  // namespace kv4
