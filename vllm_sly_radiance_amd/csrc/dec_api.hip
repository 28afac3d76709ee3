// C ABI of libdecode_ops.so: argument validation and dispatch. Declarations: include/decode_ops.h.
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

#include "decode_ops.h"
#include "dec_internal.h"

#define DEC_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace dec;

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
  if (e == hipSuccess) return DEC_OK;
  return fail(DEC_EHIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

// Sizes of a batch and its states; `step` elements: what a slot's stride is a multiple of.
int check_sequences(const char* who, const Sequences& s, long slot_elements, int step) {
  if (s.total < 0 || s.batch < 0 || s.max_q < 0)
    return fail(DEC_EINVAL, "%s: total=%d batch=%d max_q=%d", who, s.total, s.batch, s.max_q);
  if (s.slots < 0 || s.slots > 0x7FFFFFFFL) return fail(DEC_EINVAL, "%s: %ld slots", who, s.slots);
  if (s.slot_stride < slot_elements || s.slot_stride % step || s.slot_stride > (1L << 62) / (s.slots + 1))
    return fail(DEC_EINVAL, "%s: slot stride %ld is less than a slot's %ld elements, too large, or no multiple "
                "of %d", who, s.slot_stride, slot_elements, step);
  if (s.write_cols < 0 || s.write_stride < 0 || (s.batch > 1 && s.write_stride < std::max(s.write_cols, 1)))
    return fail(DEC_EINVAL, "%s: %d write slots a sequence, rows %ld apart", who, s.write_cols, s.write_stride);
  return DEC_OK;
}
int check_sequence_pointers(const char* who, const Sequences& s, const void* state) {
  if (!s.starts || !s.read || !s.write || !aligned(s.starts, 4) || !aligned(s.read, 4) || !aligned(s.write, 4))
    return fail(DEC_EINVAL, "%s: null or misaligned starts or slots", who);
  if ((!state && s.slots) || !aligned(state, 16))
    return fail(DEC_EINVAL, "%s: null state, or not 16-byte aligned", who);
  return DEC_OK;
}

int check_rows(const char* who, const char* what, const void* p, long ts, long hs) {
  if (!p) return fail(DEC_EINVAL, "%s: null %s", who, what);
  if (!aligned(p, 16) || ts % 8 || hs % 8 || ts < 0 || hs < 0)
    return fail(DEC_EINVAL, "%s: %s needs 16-byte aligned rows (strides of whole 8 elements, got %ld and %ld)",
                who, what, ts, hs);
  return DEC_OK;
}

int check_delta_sizes(const char* who, int total, int batch, int max_q, int write_cols, int k_heads, int v_heads,
                      int dk, int dv) {
  if (total < 0 || batch < 0 || max_q < 0 || write_cols < 0)
    return fail(DEC_EINVAL, "%s: total=%d batch=%d max_q=%d write_cols=%d", who, total, batch, max_q, write_cols);
  if (k_heads <= 0 || v_heads <= 0 || v_heads > 4096 || v_heads % k_heads)
    return fail(DEC_EINVAL, "%s: %d value heads over %d key heads", who, v_heads, k_heads);
  if ((dk != 64 && dk != 128) || (dv != 64 && dv != 128))
    return fail(DEC_EINVAL, "%s: heads of %d and %d channels are none of 64, 128", who, dk, dv);
  if ((long)batch * v_heads * (dv / 16) > kMaxGrid || ((long)total / kChunk + batch) * v_heads > kMaxGrid)
    return fail(DEC_EINVAL, "%s: total=%d batch=%d of %d heads is too large", who, total, batch, v_heads);
  return DEC_OK;
}

}  // namespace

DEC_API int dec_abi_version(void) { return DEC_ABI_VERSION; }
DEC_API const char* dec_last_error(void) { return g_err; }

DEC_API int dec_causal_conv(const void* x, long x_ts, const void* weight, const void* bias, void* state,
                            long slots, long slot_stride, const int* q_starts, const int* read_slots,
                            const int* write_slots, long write_stride, int write_cols, void* out, int total,
                            int batch, int max_q, int channels, int width, int flags, void* stream) {
  const char* who = "causal_conv";
  if (channels <= 0 || channels % 8 || channels > 1 << 24)
    return fail(DEC_EINVAL, "%s: %d channels: need a multiple of 8", who, channels);
  if (width < 2 || width > 4) return fail(DEC_EINVAL, "%s: width %d is none of 2, 3, 4", who, width);
  if (flags & ~DEC_SILU) return fail(DEC_EINVAL, "%s: unknown flags %d", who, flags);
  ConvArgs a = {};
  a.s = {q_starts, read_slots, write_slots, write_stride, slots, slot_stride, write_cols, total, batch, max_q};
  if (int rc = check_sequences(who, a.s, (long)(width - 1) * channels, 8)) return rc;
  if (total > 1 << 30)                  // (a lane's next run of tokens is counted in 32 bits)
    return fail(DEC_EINVAL, "%s: total=%d: need 2^30 at most", who, total);
  if ((long)batch * kv4::ceil_div(channels / 8, 256) > kMaxGrid)
    return fail(DEC_EINVAL, "%s: batch=%d of %d channels is too large", who, batch, channels);
  if (!batch) return DEC_OK;
  if (int rc = check_sequence_pointers(who, a.s, state)) return rc;
  if (!weight || !aligned(weight, 16) || !aligned(bias, 16))
    return fail(DEC_EINVAL, "%s: null weight, or weight or bias not 16-byte aligned", who);
  if (total) {
    if (int rc = check_rows(who, "x", x, x_ts, 0)) return rc;
    if (!out || !aligned(out, 16)) return fail(DEC_EINVAL, "%s: null or misaligned output", who);
  }
  a.x = (const uint16_t*)x, a.x_ts = x_ts, a.w = (const uint16_t*)weight, a.bias = (const uint16_t*)bias;
  a.state = (uint16_t*)state, a.out = (uint16_t*)out, a.C = channels, a.silu = flags & DEC_SILU;
  return hip_status(launch_conv(a, width, (hipStream_t)stream), who);
}

DEC_API int dec_gated_delta_workspace(int total, int batch, int max_q, int write_cols, int k_heads, int v_heads,
                                      int dk, int dv, size_t* bytes) {
  const char* who = "gated_delta_workspace";
  if (!bytes) return fail(DEC_EINVAL, "%s: null output", who);
  if (int rc = check_delta_sizes(who, total, batch, max_q, write_cols, k_heads, v_heads, dk, dv)) return rc;
  *bytes = batch ? delta_plan(total, batch, max_q, write_cols, k_heads, v_heads, dk, dv).workspace : 0;
  return DEC_OK;
}

DEC_API int dec_gated_delta(const void* q, long q_ts, long q_hs, const void* k, long k_ts, long k_hs,
                            const void* v, long v_ts, long v_hs, const void* a, long a_ts, const void* b,
                            long b_ts, const float* a_log, const float* dt_bias, float* state, long slots,
                            long slot_stride, const int* q_starts, const int* read_slots,
                            const int* write_slots, long write_stride, int write_cols, void* out,
                            void* workspace, size_t workspace_bytes, int total, int batch, int max_q,
                            int k_heads, int v_heads, int dk, int dv, float scale, float eps, void* stream) {
  const char* who = "gated_delta_rule";
  if (int rc = check_delta_sizes(who, total, batch, max_q, write_cols, k_heads, v_heads, dk, dv)) return rc;
  DeltaArgs d = {};
  d.s = {q_starts, read_slots, write_slots, write_stride, slots, slot_stride, write_cols, total, batch, max_q};
  if (int rc = check_sequences(who, d.s, (long)v_heads * dk * dv, 4)) return rc;
  if (!(scale == scale) || !(eps >= 0.0f))
    return fail(DEC_EINVAL, "%s: scale is NaN, or eps negative or NaN", who);
  if (!batch) return DEC_OK;
  if (int rc = check_sequence_pointers(who, d.s, state)) return rc;
  if (!a_log || !dt_bias || !aligned(a_log, 4) || !aligned(dt_bias, 4))
    return fail(DEC_EINVAL, "%s: null or misaligned a_log or dt_bias", who);
  if (total) {
    if (int rc = check_rows(who, "q", q, q_ts, q_hs)) return rc;
    if (int rc = check_rows(who, "k", k, k_ts, k_hs)) return rc;
    if (int rc = check_rows(who, "v", v, v_ts, v_hs)) return rc;
    if (v_ts > 1 << 23)                 // (rows of a chunk are counted in 32 bits)
      return fail(DEC_EINVAL, "%s: v's tokens are %ld elements apart: need 2^23 at most", who, v_ts);
    if (!a || !b || !aligned(a, 2) || !aligned(b, 2) || a_ts < 0 || b_ts < 0)
      return fail(DEC_EINVAL, "%s: null or misaligned a or b, or strides %ld and %ld", who, a_ts, b_ts);
    if (!out || !aligned(out, 16)) return fail(DEC_EINVAL, "%s: null or misaligned output", who);
  }
  const DeltaPlan plan = delta_plan(total, batch, max_q, write_cols, k_heads, v_heads, dk, dv);
  if (plan.workspace > workspace_bytes || (plan.workspace && (!workspace || !aligned(workspace, 16))))
    return fail(DEC_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", who, plan.workspace,
                workspace_bytes);
  d.q = (const uint16_t*)q, d.q_ts = q_ts, d.q_hs = q_hs;
  d.k = (const uint16_t*)k, d.k_ts = k_ts, d.k_hs = k_hs;
  d.v = (const uint16_t*)v, d.v_ts = v_ts, d.v_hs = v_hs;
  d.a = (const uint16_t*)a, d.a_ts = a_ts, d.b = (const uint16_t*)b, d.b_ts = b_ts;
  d.a_log = a_log, d.dt_bias = dt_bias, d.state = state, d.out = (uint16_t*)out, d.workspace = workspace;
  d.Hk = k_heads, d.Hv = v_heads, d.scale = scale, d.eps = eps;
  if (plan.chunks) {
    d.keys = plan.keys;
    return hip_status(launch_delta_chunks(d, dk, dv, (hipStream_t)stream), who);
  }
  return hip_status(launch_delta_steps(d, dk, dv, (hipStream_t)stream), who);
}

namespace {
int check_sample_sizes(const char* who, int rows, int vocabulary, int flags) {
  if (rows < 0 || rows > 1 << 21) return fail(DEC_EINVAL, "%s: %d rows", who, rows);
  if (vocabulary <= 0 || vocabulary > 1 << 24)
    return fail(DEC_EINVAL, "%s: a vocabulary of %d: need 1..2^24", who, vocabulary);
  if (flags & ~(DEC_BF16 | DEC_LOGPROBS)) return fail(DEC_EINVAL, "%s: unknown flags %d", who, flags);
  return DEC_OK;
}
}  // namespace

DEC_API int dec_sample_workspace(int rows, int vocabulary, int top_k, int flags, size_t* bytes) {
  const char* who = "sample_workspace";
  if (!bytes) return fail(DEC_EINVAL, "%s: null output", who);
  if (int rc = check_sample_sizes(who, rows, vocabulary, flags)) return rc;
  *bytes = sample_workspace(rows, sample_parts(rows, vocabulary, flags & DEC_BF16, top_k));
  return DEC_OK;
}

DEC_API int dec_sample(const void* logits, long row_stride, const float* uniform, const float* temperature,
                       float temperature_all, const int* top_k, int top_k_all, const float* top_p,
                       float top_p_all, const float* min_p, float min_p_all, int64_t* tokens, float* logprobs,
                       void* workspace, size_t workspace_bytes, int rows, int vocabulary, int flags,
                       void* stream) {
  const char* who = "sample";
  if (int rc = check_sample_sizes(who, rows, vocabulary, flags)) return rc;
  const int size = flags & DEC_BF16 ? 2 : 4;
  if (rows > 1 && row_stride < vocabulary)
    return fail(DEC_EINVAL, "%s: rows %ld apart for a vocabulary of %d", who, row_stride, vocabulary);
  if (!rows) return DEC_OK;
  if (!logits || !aligned(logits, size) || !uniform || !aligned(uniform, 4))
    return fail(DEC_EINVAL, "%s: null or misaligned logits or uniform numbers", who);
  if (!aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4))
    return fail(DEC_EINVAL, "%s: misaligned parameters", who);
  if (!tokens || !aligned(tokens, 8) || ((flags & DEC_LOGPROBS) && (!logprobs || !aligned(logprobs, 4))))
    return fail(DEC_EINVAL, "%s: null or misaligned output", who);
  const int parts = sample_parts(rows, vocabulary, flags & DEC_BF16, top_k ? 1 : top_k_all);
  const size_t need = sample_workspace(rows, parts);
  if (need > workspace_bytes || (need && (!workspace || !aligned(workspace, 16))))
    return fail(DEC_EINVAL, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", who, need, workspace_bytes);
  SampleArgs a = {};
  a.logits = logits, a.uniform = uniform, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p;
  a.min_p = min_p, a.tokens = tokens, a.logprobs = flags & DEC_LOGPROBS ? logprobs : nullptr;
  a.workspace = workspace, a.parts = parts;
  a.row_stride = rows > 1 ? row_stride : 0, a.rows = rows, a.V = vocabulary;
  a.temperature_all = temperature_all, a.top_k_all = top_k_all, a.top_p_all = top_p_all, a.min_p_all = min_p_all;
  a.bf16 = flags & DEC_BF16;
  return hip_status(launch_sample(a, (hipStream_t)stream), who);
}
