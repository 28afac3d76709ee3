/* C ABI of the MI355X (gfx950) operators of a hybrid decoder beside its projections and its
 * attention, libdecode_ops.so: the short causal convolution and the gated delta rule of its
 * linear-attention layers, and the choice of its next tokens.
 *
 * Plain pointers, sizes and a HIP stream (as void*); no torch or C++ types cross this boundary.
 * Device pointers are HIP device addresses owned by the caller; the library never allocates device
 * memory. Launches are asynchronous on the given stream, so they are HIP-graph-capture safe. Every
 * entry point validates its arguments before launching anything and returns DEC_OK (0) or a nonzero
 * status that dec_last_error() describes (thread-local). What only the device knows (starts, slots,
 * what the rows of logits hold) is checked by the kernels, which never leave the buffers they are
 * given.
 *
 * Sequences. The tokens of a batch lie one sequence after the other: sequence b's are rows
 * q_starts[b] .. q_starts[b + 1] - 1 of `total` (int32 [batch + 1]). max_q, at least the most tokens
 * of a sequence, chooses the form of the work only. Rows that no sequence owns are not written;
 * starts that go back leave outputs and states unspecified.
 *
 * States. A sequence goes on from the state in slot read_slots[b] (int32 [batch]): from zeros where
 * that is negative, from NaN where it is past the slots. Its new state goes to write_slots, int32
 * [batch][write_cols] with rows write_stride apart. write_cols = 0 (one number a sequence): the state
 * after its last token (the one read where it has none). write_cols > 0: the state after token i to
 * slot write_slots[b][i], for i < write_cols. Negative slots and those past the end are not written. A
 * slot that one sequence writes may be read by that sequence only, and written by one only.
 */
#ifndef DECODE_OPS_H_
#define DECODE_OPS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DEC_ABI_VERSION 1

enum {
  DEC_OK = 0,
  DEC_EINVAL = 1, /* bad shape, pointer, stride or alignment */
  DEC_EHIP = 3    /* the HIP runtime reported an error at launch */
};

/* Bits of the `flags` arguments. */
enum {
  DEC_SILU = 1,    /* causal_conv: SiLU of the sums */
  DEC_BF16 = 2,    /* sample: logits are bf16 instead of fp32 */
  DEC_LOGPROBS = 4 /* sample: log probabilities too */
};

/* ABI version of the loaded library (DEC_ABI_VERSION). */
int dec_abi_version(void);

/* Description of this thread's most recent failing call. */
const char* dec_last_error(void);

/* Depthwise causal convolution of `width` 2, 3 or 4 over each sequence's tokens, `total` 2^30 at most:
 *   out[t][c] = f(bias[c] + sum_i weight[c][i] x[t - width + 1 + i][c]), f SiLU or nothing,
 * in fp32, rounded once. x bf16 [total][channels] with rows x_ts elements apart (16-byte aligned, x_ts
 * and channels multiples of 8); weight bf16 [channels][width] and bias bf16 [channels] (or null),
 * 16-byte aligned; out bf16 [total][channels]. What lies before the first token is the state, bf16
 * [slots][width - 1][channels], slots slot_stride elements apart (a multiple of 8): the last width - 1
 * inputs, oldest first. */
int dec_causal_conv(const void* x, long x_ts, const void* weight, const void* bias, void* state,
                    long slots, long slot_stride, const int* q_starts, const int* read_slots,
                    const int* write_slots, long write_stride, int write_cols, void* out, int total,
                    int batch, int max_q, int channels, int width, int flags, void* stream);

/* The gated delta rule. For each sequence and value head, token after token, with the state S
 * [dk][dv] in fp32:
 *   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  out = scale S^T q
 * with q and k divided by sqrt(sum of squares + eps), g = -exp(a_log) softplus(a + dt_bias) and beta =
 * sigmoid(b). q, k bf16 [total][k_heads][dk] and v bf16 [total][v_heads][dv] (16-byte aligned; strides
 * of tokens *_ts and heads *_hs multiples of 8 elements); value head h takes key head h / (v_heads /
 * k_heads). a, b bf16 [total][v_heads], tokens a_ts and b_ts elements apart; a_log, dt_bias fp32
 * [v_heads]. state fp32 [slots][v_heads][dk][dv], slots slot_stride elements apart (a multiple of 4),
 * 16-byte aligned. out bf16 [total][v_heads][dv]. dk and dv: 64 or 128. `workspace`:
 * dec_gated_delta_workspace bytes, 16-byte aligned, the call's own until it has run: none with max_q 16 at most or
 * write_cols > 0, else 25600 a value head and 49152 a key head (24576 with dk 64) for each of total / 64 + batch chunks, 31
 * KB a token of 48 and 16 heads. */
int dec_gated_delta(const void* q, long q_ts, long q_hs, const void* k, long k_ts, long k_hs,
                    const void* v, long v_ts, long v_hs, const void* a, long a_ts, const void* b,
                    long b_ts, const float* a_log, const float* dt_bias, float* state, long slots,
                    long slot_stride, const int* q_starts, const int* read_slots,
                    const int* write_slots, long write_stride, int write_cols, void* out,
                    void* workspace, size_t workspace_bytes, int total, int batch, int max_q,
                    int k_heads, int v_heads, int dk, int dv, float scale, float eps, void* stream);
int dec_gated_delta_workspace(int total, int batch, int max_q, int write_cols, int k_heads, int v_heads,
                              int dk, int dv, size_t* bytes);

/* One token of each row of logits (fp32, or bf16 with DEC_BF16; rows row_stride elements apart). With
 * top = max x, t = temperature, w_i = 1 where x_i = top, 0 where x_i = -infinity, else exp((x_i - top) / t)
 * in 64 bits, and the row in descending order of x, ties by index:
 *   the first top_k of the order; of those the shortest prefix whose sum of w is at least top_p times
 *   theirs (one token at least); of those the ones with w >= min_p (the first in any case).
 * The token is the lowest index at which the sum of the kept w up to it exceeds uniform times their sum
 * (uniform held to [0, 1); NaN counts as 0). t <= 0: the first in the order. top_k < 1 or past the
 * vocabulary, top_p >= 1 or NaN, min_p <= 0 or NaN filter nothing. A row that holds NaN or nothing above
 * -infinity, and one whose t is NaN, gives token -1 and log probability NaN. Weights are added as
 * integers of 2^-min(51, 62 - ceil(log2 vocabulary)), so that results do not depend on an order of additions.
 * temperature fp32, top_k int32, top_p fp32, min_p fp32 [rows], or null: the value *_all for all rows.
 * uniform fp32 [rows]; tokens int64 [rows]; logprobs (DEC_LOGPROBS) fp32 [rows], of the softmax of the
 * logits as they are (no temperature, no filter). `workspace`: dec_sample_workspace bytes (top_k: the value
 * for all rows, or 1 where they have their own), 16-byte aligned, the call's own until it has run. */
int dec_sample(const void* logits, long row_stride, const float* uniform, const float* temperature,
               float temperature_all, const int* top_k, int top_k_all, const float* top_p,
               float top_p_all, const float* min_p, float min_p_all, int64_t* tokens, float* logprobs,
               void* workspace, size_t workspace_bytes, int rows, int vocabulary, int flags,
               void* stream);
int dec_sample_workspace(int rows, int vocabulary, int top_k, int flags, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif
