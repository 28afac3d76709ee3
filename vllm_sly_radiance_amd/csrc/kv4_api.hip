// C ABI of libkv4_attn.so: argument validation and dispatch. Declarations: include/kv4_attn.h.
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <new>
#include <vector>

#include "kv4_attn.h"
#include "kv4_internal.h"

#define KV4_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace kv4;

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int hip_status(hipError_t e, const char* what) {
  if (e == hipSuccess) return KV4_OK;
  return fail(KV4_EHIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Workgroups of 256 threads that one launch may have: its threads are counted in 32 bits.
constexpr long kMaxGrid = (1L << 32) / 256 - 1;

int check_heads(const char* who, int heads, int d) {
  if (heads <= 0 || heads > 4096)
    return fail(KV4_EINVAL, "%s: need 1..4096 heads, got %d", who, heads);
  if (d != 64 && d != 128 && d != 256)
    return fail(KV4_EINVAL, "%s: head size %d is none of 64, 128, 256", who, d);
  return KV4_OK;
}

int page_shift(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

int check_cache(const char* who, const void* cache, long pages, long page_stride, int page,
                int heads, int d) {
  if (page_shift(page) < 0)
    return fail(KV4_EINVAL, "%s: page of %d tokens is none of 16, 32, 64, 128, 256", who, page);
  if (pages < 0 || pages > 0x7FFFFFFFL)
    return fail(KV4_EINVAL, "%s: %ld pages", who, pages);
  const long bytes = (long)heads * (page / 16) * 17 * d;
  if (page_stride < bytes || page_stride % 16 || page_stride >> 32)
    return fail(KV4_EINVAL, "%s: page stride %ld is less than a page's %ld bytes, 2^32 or more, or no "
                "multiple of 16", who, page_stride, bytes);
  if (!cache && pages) return fail(KV4_EINVAL, "%s: null cache", who);
  if (!aligned(cache, 16)) return fail(KV4_EINVAL, "%s: the cache is not 16-byte aligned", who);
  return KV4_OK;
}

int check_rows(const char* who, const char* what, const void* p, long ts, long hs) {
  if (!p) return fail(KV4_EINVAL, "%s: null %s", who, what);
  if (!aligned(p, 16) || ts % 8 || hs % 8 || ts < 0 || hs < 0)
    return fail(KV4_EINVAL,
                "%s: %s needs 16-byte aligned heads (strides of whole 8 elements, got %ld and %ld)",
                who, what, ts, hs);
  return KV4_OK;
}

int rope(const char* who, RopeArgs a, int q_heads, int kv_heads, int d, hipStream_t stream) {
  if (a.T < 0) return fail(KV4_EINVAL, "%s: T=%d", who, a.T);
  if (int rc = check_heads(who, q_heads, d)) return rc;
  if (int rc = check_heads(who, kv_heads, d)) return rc;
  if (a.rot < 0 || a.rot > d || a.rot % 16)
    return fail(KV4_EINVAL, "%s: %d rotated channels: need a multiple of 16 up to the head size %d",
                who, a.rot, d);
  if (a.rot && (a.axes < 1 || (a.axes > 1 && !a.axis)))
    return fail(KV4_EINVAL, "%s: %d position axes%s", who, a.axes,
                a.axes > 1 ? " need the axis of each pair" : "");
  if (a.flags & ~(KV4_PLUS_ONE | KV4_ADJACENT | KV4_TABLE_BF16 | KV4_POS_I32))
    return fail(KV4_EINVAL, "%s: unknown flags %d", who, a.flags);
  if (a.T == 0) return KV4_OK;
  if (int rc = check_rows(who, "q", a.q.p, a.q.ts, a.q.hs)) return rc;
  if (int rc = check_rows(who, "k", a.k.p, a.k.ts, a.k.hs)) return rc;
  if (!aligned(a.qw, 16) || !aligned(a.kw, 16))
    return fail(KV4_EINVAL, "%s: the norm weights need 16-byte alignment", who);
  if (a.rot) {
    if (!a.table || !a.pos || a.rows < 0)
      return fail(KV4_EINVAL, "%s: null table or positions, or %ld table rows", who, a.rows);
    if (!aligned(a.table, a.flags & KV4_TABLE_BF16 ? 2 : 4) || !aligned(a.axis, 4) ||
        !aligned(a.pos, a.flags & KV4_POS_I32 ? 4 : 8))
      return fail(KV4_EINVAL, "%s: misaligned table, positions or axes", who);
    if (a.pos_stride < 0 || (a.axes > 1 && a.pos_stride < a.T))
      return fail(KV4_EINVAL, "%s: position rows of %ld for %d tokens", who, a.pos_stride, a.T);
  }
  if (!a.q_out || !aligned(a.q_out, 16) || (!a.cache && (!a.k_out || !aligned(a.k_out, 16))))
    return fail(KV4_EINVAL, "%s: null or misaligned output", who);
  if ((long)a.T * (q_heads + 2 * kv_heads) > 4 * kMaxGrid)
    return fail(KV4_EINVAL, "%s: T=%d is too large", who, a.T);
  return hip_status(launch_rope(a, d, stream), who);
}

// Checks the sizes of an attention call and plans it (an empty plan where there is nothing to do).
int plan_attention(const char* who, int total, int batch, int max_q, int max_len, int q_heads,
                   int kv_heads, int d, int window, AttnPlan* plan) {
  if (int rc = check_heads(who, kv_heads, d)) return rc;
  if (int rc = check_heads(who, q_heads, d)) return rc;
  if (q_heads % kv_heads)
    return fail(KV4_EINVAL, "%s: %d query heads over %d kv heads", who, q_heads, kv_heads);
  if (batch < 0 || max_q < 0 || max_len < 0 || max_len > 0x7FFFF000 || window < 0)
    return fail(KV4_EINVAL, "%s: batch=%d max_q=%d max_len=%d window=%d", who, batch, max_q, max_len,
                window);
  // what the counts below need to be exact: rows at the limits, and row tiles of 16 of them, which is
  // what the kernels count in 32 bits whatever the starts on the device are
  const long heads = (long)batch * q_heads, rows = (long)std::min(max_q, std::max(total, 0)) * q_heads;
  if ((max_q && heads > (1L << 40) / max_q) || rows > 0x7FFFF000L ||
      batch * (rows / 16 + kv_heads) > 0x7FFFFFFFL)
    return fail(KV4_EINVAL, "%s: batch=%d max_q=%d q_heads=%d are too many rows", who, batch, max_q,
                q_heads);
  *plan = {};
  if (total <= 0 || !batch) return KV4_OK;
  // (where no sequence may have queries, those that do are written as NaN: planned as for one each)
  *plan = attn_plan(total, batch, std::max(std::min(max_q, total), 1), max_len, q_heads, kv_heads, d, window);
  // attn_rows counts its work in 31 bits, a launch its threads in 32
  if (plan->work > 0x7FFFFFFFL - 4 * kCUs || plan->threads >> 32)
    return fail(KV4_EINVAL, "%s: batch=%d total=%d max_len=%d are too much for one call", who, batch, total,
                max_len);
  return KV4_OK;
}

}  // namespace

KV4_API int kv4_abi_version(void) { return KV4_ABI_VERSION; }
KV4_API const char* kv4_last_error(void) { return g_err; }

KV4_API int kv4_page_bytes(int heads, int page, int d, size_t* bytes) {
  if (!bytes) return fail(KV4_EINVAL, "page_bytes: null output");
  if (int rc = check_heads("page_bytes", heads, d)) return rc;
  if (page_shift(page) < 0)
    return fail(KV4_EINVAL, "page_bytes: page of %d tokens is none of 16, 32, 64, 128, 256", page);
  *bytes = (size_t)heads * (page / 16) * 17 * d;
  return KV4_OK;
}

KV4_API int kv4_qk_norm_rope(const void* q, long q_ts, long q_hs, const void* k, long k_ts, long k_hs,
                             const void* q_weight, const void* k_weight, const void* cos_sin,
                             long table_rows, int rot, const void* positions, long pos_stride,
                             int axes, const int* axis_of_pair, void* q_out, void* k_out, int T,
                             int q_heads, int kv_heads, int d, float eps, int flags, void* stream) {
  RopeArgs a = {};
  a.q = {(const uint16_t*)q, q_ts, q_hs};
  a.k = {(const uint16_t*)k, k_ts, k_hs};
  a.qw = (const uint16_t*)q_weight, a.kw = (const uint16_t*)k_weight;
  a.table = cos_sin, a.rows = table_rows, a.rot = rot;
  a.pos = positions, a.pos_stride = pos_stride, a.axes = axes, a.axis = axis_of_pair;
  a.q_out = (uint16_t*)q_out, a.k_out = (uint16_t*)k_out;
  a.T = T, a.Hq = q_heads, a.Hkv = kv_heads, a.eps = eps, a.flags = flags;
  a.page_shift = 4;
  return rope("qk_norm_rope", a, q_heads, kv_heads, d, (hipStream_t)stream);
}

KV4_API int kv4_qk_norm_rope_append(const void* q, long q_ts, long q_hs, const void* k, long k_ts,
                                    long k_hs, const void* v, long v_ts, long v_hs,
                                    const void* q_weight, const void* k_weight, const void* cos_sin,
                                    long table_rows, int rot, const void* positions, long pos_stride,
                                    int axes, const int* axis_of_pair, void* q_out, void* cache,
                                    long pages, long page_stride, int page, const int64_t* slots,
                                    int T, int q_heads, int kv_heads, int d, float eps, int flags,
                                    void* stream) {
  const char* who = "qk_norm_rope_append";
  if (int rc = check_heads(who, kv_heads, d)) return rc;
  if (int rc = check_cache(who, cache, pages, page_stride, page, kv_heads, d)) return rc;
  if (T > 0) {
    if (!cache) return fail(KV4_EINVAL, "%s: null cache", who);
    if (!slots || !aligned(slots, 8)) return fail(KV4_EINVAL, "%s: null or misaligned slots", who);
    if (int rc = check_rows(who, "v", v, v_ts, v_hs)) return rc;
  }
  RopeArgs a = {};
  a.q = {(const uint16_t*)q, q_ts, q_hs};
  a.k = {(const uint16_t*)k, k_ts, k_hs};
  a.v = {(const uint16_t*)v, v_ts, v_hs};
  a.qw = (const uint16_t*)q_weight, a.kw = (const uint16_t*)k_weight;
  a.table = cos_sin, a.rows = table_rows, a.rot = rot;
  a.pos = positions, a.pos_stride = pos_stride, a.axes = axes, a.axis = axis_of_pair;
  a.q_out = (uint16_t*)q_out;
  a.cache = (uint8_t*)cache, a.slots = slots, a.pages = pages, a.page_stride = page_stride;
  a.page_shift = page_shift(page);
  a.T = T, a.Hq = q_heads, a.Hkv = kv_heads, a.eps = eps, a.flags = flags;
  return rope(who, a, q_heads, kv_heads, d, (hipStream_t)stream);
}

KV4_API int kv4_gather(const void* cache, long pages, long page_stride, int page,
                       const int64_t* slots, void* k, void* v, int T, int heads, int d,
                       void* stream) {
  const char* who = "gather";
  if (T < 0) return fail(KV4_EINVAL, "%s: T=%d", who, T);
  if (int rc = check_heads(who, heads, d)) return rc;
  if (int rc = check_cache(who, cache, pages, page_stride, page, heads, d)) return rc;
  if (T == 0) return KV4_OK;
  if (!slots || !aligned(slots, 8)) return fail(KV4_EINVAL, "%s: null or misaligned slots", who);
  if (!k || !v || !aligned(k, 16) || !aligned(v, 16))
    return fail(KV4_EINVAL, "%s: null or misaligned output", who);
  if ((long)T * heads > 0x7FFFFFFFL || (long)T * heads * (d / 8) / 256 > kMaxGrid)
    return fail(KV4_EINVAL, "%s: T=%d is too large", who, T);
  GatherArgs a = {(const uint8_t*)cache, slots, (uint16_t*)k, (uint16_t*)v, pages, page_stride,
                  page_shift(page), T, heads};
  return hip_status(launch_gather(a, d, (hipStream_t)stream), who);
}

KV4_API int kv4_attention_workspace(int total, int batch, int max_q, int max_len, int q_heads,
                                    int kv_heads, int d, int window, size_t* bytes) {
  if (!bytes) return fail(KV4_EINVAL, "attention_workspace: null output");
  AttnPlan plan;
  if (int rc = plan_attention("attention_workspace", total, batch, max_q, max_len, q_heads, kv_heads, d,
                              window, &plan))
    return rc;
  *bytes = plan.workspace;
  return KV4_OK;
}

KV4_API int kv4_attention(const void* q, long q_ts, long q_hs, const void* cache, long pages,
                          long page_stride, int page, const int* page_table, long table_stride,
                          int table_cols, const int* seq_lens, const int* q_starts, void* out,
                          void* workspace, size_t workspace_bytes, int total, int batch, int max_q,
                          int max_len, int q_heads, int kv_heads, int d, float scale, int window,
                          int flags, void* stream) {
  const char* who = "attention";
  AttnPlan plan;
  if (int rc = plan_attention(who, total, batch, max_q, max_len, q_heads, kv_heads, d, window, &plan))
    return rc;
  if (int rc = check_cache(who, cache, pages, page_stride, page, kv_heads, d)) return rc;
  if (!(scale > 0.0f) || scale > 3.0e38f)
    return fail(KV4_EINVAL, "%s: scale must be positive and finite", who);
  if (flags & ~KV4_CAUSAL) return fail(KV4_EINVAL, "%s: unknown flags %d", who, flags);
  if (total < 0 || table_cols < 0 || table_stride < 0)
    return fail(KV4_EINVAL, "%s: total=%d table_cols=%d table_stride=%ld", who, total, table_cols,
                table_stride);
  if (!total || !batch) return KV4_OK;
  if (int rc = check_rows(who, "q", q, q_ts, q_hs)) return rc;
  if (!seq_lens || !q_starts || (!page_table && table_cols) || !out)
    return fail(KV4_EINVAL, "%s: null pointer", who);
  if (!aligned(seq_lens, 4) || !aligned(q_starts, 4) || !aligned(page_table, 4) || !aligned(out, 16))
    return fail(KV4_EINVAL, "%s: misaligned pointer", who);
  if (plan.workspace > workspace_bytes || (plan.workspace && (!workspace || !aligned(workspace, 16))))
    return fail(KV4_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", who,
                plan.workspace, workspace_bytes);
  AttnArgs a = {};
  a.q = (const uint16_t*)q, a.cache = (const uint8_t*)cache, a.pages_of = page_table;
  a.lens = seq_lens, a.starts = q_starts, a.out = (uint16_t*)out, a.part = (float*)workspace;
  a.q_ts = q_ts, a.q_hs = q_hs, a.page_stride = page_stride, a.pages = pages;
  a.table_stride = table_stride, a.page_shift = page_shift(page);
  // An unusable page is read as page 0, which a cache of no pages does not have: no token of it has a
  // page, so that every sequence with tokens is longer than its row of the table (NaN).
  a.table_cols = pages ? table_cols : 0;
  a.total = total, a.batch = batch, a.max_len = max_len;
  a.max_q = std::min(max_q, total);     // (a sequence of more queries than rows is bad either way)
  a.Hq = q_heads, a.Hkv = kv_heads, a.group = q_heads / kv_heads;
  a.window = window, a.scale = scale;
  a.causal = flags & KV4_CAUSAL;
  a.few_rows = plan.few_rows;
  if (plan.tiles) {
    a.units = plan.units, a.entries = plan.entries, a.span = plan.span;
    if (int rc = hip_status(launch_attn_tiles(a, d, (hipStream_t)stream), who)) return rc;
    a.entries = 0, a.part += plan.tiles_workspace / sizeof(float);
  }
  a.fragments = plan.fragments, a.runs = plan.runs;
  return plan.rows ? hip_status(launch_attn_rows(a, d, (hipStream_t)stream), who) : KV4_OK;
}

KV4_API int kv4_move_pages(void* cache, int layers, long layer_stride, long pages, long page_stride,
                           size_t page_bytes, const int* pairs, int n, int* tables, int table_rows,
                           int table_cols, long table_stride, void* stream) {
  const char* who = "move_pages";
  if (n < 0 || layers < 0 || pages < 0 || pages > 0x7FFFFFFFL)
    return fail(KV4_EINVAL, "%s: n=%d layers=%d pages=%ld", who, n, layers, pages);
  if (page_bytes % 16 || page_stride % 16 || layer_stride % 16 || page_stride < 0 || layer_stride < 0 ||
      (size_t)page_stride < page_bytes)
    return fail(KV4_EINVAL, "%s: page bytes and strides are multiples of 16, a page stride at least "
                "the page (got %zu, %ld, %ld)", who, page_bytes, page_stride, layer_stride);
  if (n && !pairs) return fail(KV4_EINVAL, "%s: null pairs", who);
  if (n && layers && page_bytes && (!cache || !aligned(cache, 16)))
    return fail(KV4_EINVAL, "%s: null or misaligned cache", who);
  if (tables && (table_rows < 0 || table_cols < 0 || !aligned(tables, 4) ||
                 (table_rows > 1 && table_stride < table_cols)))
    return fail(KV4_EINVAL, "%s: page table of %d x %d with row stride %ld", who, table_rows,
                table_cols, table_stride);
  if (n > pages) return fail(KV4_EINVAL, "%s: %d pairs over %ld pages", who, n, pages);
  try {
    std::vector<std::pair<int, int>> list(n);
    std::vector<int> to(n);
    for (int i = 0; i < n; ++i) {
      const int s = pairs[2 * i], d = pairs[2 * i + 1];
      if (s < 0 || s >= pages || d < 0 || d >= pages)
        return fail(KV4_EINVAL, "%s: pair %d (%d -> %d) is outside the %ld pages", who, i, s, d, pages);
      list[i] = {s, d}, to[i] = d;
    }
    std::sort(list.begin(), list.end());
    std::sort(to.begin(), to.end());
    for (int i = 1; i < n; ++i) {
      if (to[i] == to[i - 1]) return fail(KV4_EINVAL, "%s: page %d is written twice", who, to[i]);
      if (tables && list[i].first == list[i - 1].first)
        return fail(KV4_EINVAL, "%s: page %d has two places in the page table", who, list[i].first);
    }
    for (int i = 0; i < n; ++i)
      if (std::binary_search(to.begin(), to.end(), list[i].first))
        return fail(KV4_EINVAL, "%s: page %d is both read and written", who, list[i].first);
    MoveArgs a = {(uint8_t*)cache, layer_stride, page_stride, page_bytes, tables, table_stride,
                  layers, table_rows, table_cols};
    for (int at = 0; at < n; at += kMovePairs) {
      const int m = std::min(kMovePairs, n - at);
      const long parts = (long)((page_bytes + 16383) / 16384);
      if (parts * m * layers + ((long)table_rows * table_cols + 255) / 256 > kMaxGrid)
        return fail(KV4_EINVAL, "%s: %d pages of %zu bytes in %d layers are too much for one call",
                    who, n, page_bytes, layers);
      int flat[2 * kMovePairs];
      for (int i = 0; i < m; ++i)
        flat[2 * i] = list[at + i].first, flat[2 * i + 1] = list[at + i].second;
      if (int rc = hip_status(launch_move(a, flat, m, (hipStream_t)stream), who)) return rc;
    }
  } catch (const std::bad_alloc&) {
    return fail(KV4_EINVAL, "%s: out of host memory for %d pairs", who, n);
  }
  return KV4_OK;
}
