// Reading tokens back from the 4-bit cache, and moving its pages, for gfx950. Both only move bytes:
// HBM bounds them where there is enough to move (600 pages of 24 layers moved, 501 MB: 107 us, 4.7 TB/s of
// the 5.1 that a large copy reaches; 4096 tokens of 16 heads of 128 read back, 43 MB: 11.6 us, 3.7 TB/s, with
// one item a lane in flight, whose codes and scales wait for its slot), launch latency where there is not (61
// tokens 2.8 us, 4 pages of 24 layers 3.2).
#include "kv4_attn.h"
#include "kv4_internal.h"

namespace kv4 {
namespace {

// One lane per 8 channels of a token's head, as the append kernel writes them: 4 bytes of codes and
// one scale byte (4 lanes share it) to 16 bytes of bf16, keys and values.
template <int D>
__global__ __launch_bounds__(256) void gather_tokens(GatherArgs a, long items) {
  using G = Group<D>;
  constexpr int kLanes = D / 8;
  const long item = (long)blockIdx.x * 256 + threadIdx.x;
  if (item >= items) return;
  const int j = (int)(item & (kLanes - 1));
  const int th = (int)(item / kLanes);  // token-major: [T][H]
  const int t = a.by_heads(th), h = th - t * a.H;
  const long slot = a.slots[t];
  const long page = slot >> a.page_shift;
  const size_t at = (size_t)th * D + 8 * j;
  uint4 k, v;
  if (slot < 0 || page >= a.pages) {
    const uint32_t fill = slot < 0 ? 0u : 0x7FC07FC0u;
    k = v = make_uint4(fill, fill, fill, fill);
  } else {
    const int place = (int)(slot & ((1 << a.page_shift) - 1));
    const int token = place & 15;
    const uint8_t* group = a.cache + (size_t)page * a.page_stride +
                           ((size_t)h << (a.page_shift - 4)) * G::kBytes +
                           (size_t)(place >> 4) * G::kBytes;
    const uint32_t kc =
        *reinterpret_cast<const uint32_t*>(group + G::kKeys + token * (D / 2) + 4 * j);
    const float ks = stored_scale(group[G::kKeyScales + token * (D / kBlock) + (j >> 2)]);
    const float vs = stored_scale(group[G::kValueScales + (j >> 2) * kGroup + token]);
    const int g = token >> 2, i = token & 3;
    uint32_t vc;
    if constexpr (G::kRun == 8) {
      vc = *reinterpret_cast<const uint32_t*>(
          group + G::kValues + ((((j >> 4) * 4 + g) * 16 + (j & 15)) * 4 + i) * 4);
    } else {
      const uint8_t* p = group + G::kValues + ((g * 16 + 2 * j) * 4 + i) * 2;
      vc = *reinterpret_cast<const uint16_t*>(p) |
           (uint32_t) * reinterpret_cast<const uint16_t*>(p + 8) << 16;
    }
    k = make_uint4(codes_bf16x2<0>(kc, ks), codes_bf16x2<1>(kc, ks), codes_bf16x2<2>(kc, ks),
                   codes_bf16x2<3>(kc, ks));
    v = make_uint4(codes_bf16x2<0>(vc, vs), codes_bf16x2<1>(vc, vs), codes_bf16x2<2>(vc, vs),
                   codes_bf16x2<3>(vc, vs));
  }
  *reinterpret_cast<uint4*>(a.k + at) = k;
  *reinterpret_cast<uint4*>(a.v + at) = v;
}

template <int D>
hipError_t launch_g(GatherArgs a, hipStream_t stream) {
  a.by_heads = divisor(a.H);
  const long items = (long)a.T * a.H * (D / 8);
  gather_tokens<D><<<(unsigned)((items + 255) / 256), 256, 0, stream>>>(a, items);
  return hipGetLastError();
}

// The pairs ride in the kernel's arguments: no copy of a list to the device and nothing to keep
// alive. Workgroups [0, copies) copy kMoveBytes of one page of one layer each; the rest remap the
// table, each entry by a binary search among the sources (sorted).
template <int N>
struct Pairs { int v[N][2]; };
constexpr int kMoveBytes = 256 * 16 * 4;   // of a workgroup: four 16-byte loads a thread in flight

template <int N>
__global__ __launch_bounds__(256) void move_pages(MoveArgs a, int n, int parts, int copies,
                                                  Pairs<N> pairs) {
  const int b = blockIdx.x;
  if (b < copies) {
    const int part = b % parts, rest = b / parts;
    const int pair = rest % n, layer = rest / n;
    uint8_t* base = a.cache + (size_t)layer * a.layer_stride;
    const uint8_t* src = base + (size_t)pairs.v[pair][0] * a.page_stride;
    uint8_t* dst = base + (size_t)pairs.v[pair][1] * a.page_stride;
    const size_t at = (size_t)part * kMoveBytes + threadIdx.x * 16;
    v4i x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * 4096 < a.page_bytes)
        x[i] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(src + at + i * 4096));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * 4096 < a.page_bytes)
        __builtin_nontemporal_store(x[i], reinterpret_cast<v4i*>(dst + at + i * 4096));
    return;
  }
  __shared__ int2 list[N];
  for (int i = threadIdx.x; i < n; i += 256) list[i] = make_int2(pairs.v[i][0], pairs.v[i][1]);
  __syncthreads();
  const long entry = (long)(b - copies) * 256 + threadIdx.x;
  if (entry >= (long)a.table_rows * a.table_cols) return;
  int* p = a.tables + (entry / a.table_cols) * a.table_stride + entry % a.table_cols;
  const int page = *p;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid].x < page) lo = mid + 1;
    else hi = mid;
  }
  if (lo < n && list[lo].x == page) *p = list[lo].y;
}

template <int N>
hipError_t launch_m(const MoveArgs& a, const int* pairs, int n, hipStream_t stream) {
  Pairs<N> p;
  for (int i = 0; i < n; ++i) p.v[i][0] = pairs[2 * i], p.v[i][1] = pairs[2 * i + 1];
  for (int i = n; i < N; ++i) p.v[i][0] = p.v[i][1] = 0;
  const int parts = (int)((a.page_bytes + kMoveBytes - 1) / kMoveBytes);
  const int copies = parts * n * a.layers;
  const long entries = a.tables ? (long)a.table_rows * a.table_cols : 0;
  move_pages<N><<<(unsigned)(copies + (entries + 255) / 256), 256, 0, stream>>>(a, n, parts, copies,
                                                                                p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gather(const GatherArgs& a, int d, hipStream_t stream) {
  return d == 64 ? launch_g<64>(a, stream)
                 : d == 128 ? launch_g<128>(a, stream) : launch_g<256>(a, stream);
}

hipError_t launch_move(const MoveArgs& a, const int* pairs, int n, hipStream_t stream) {
  return n <= 16 ? launch_m<16>(a, pairs, n, stream) : launch_m<kMovePairs>(a, pairs, n, stream);
}

}  // namespace kv4
