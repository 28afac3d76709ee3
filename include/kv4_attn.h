/* C ABI of the MI355X (gfx950) attention operators over a 4-bit paged cache, libkv4_attn.so.
 *
 * What lies between a decoder's qkv and output projections: per-head RMSNorm of queries and keys
 * with the rotation, the same with the new keys and values rounded into their cache slots, softmax
 * attention over the cached tokens, reading tokens back, and moving pages.
 *
 * Plain pointers, sizes and a HIP stream (as void*); no torch or C++ types cross this boundary.
 * Device pointers are HIP device addresses owned by the caller; the library never allocates device
 * memory. Launches are asynchronous on the given stream, so they are HIP-graph-capture safe. Every
 * entry point validates its arguments before launching anything and returns KV4_OK (0) or a nonzero
 * status that kv4_last_error() describes (thread-local). What only the device knows (positions,
 * slots, page numbers, lengths) is checked by the kernels, which never leave the buffers they are
 * given: an unusable position or page gives NaN outputs for its token, a slot outside the cache is
 * not written.
 *
 * The cache. Pages of `page` tokens (16, 32, 64, 128 or 256), each [kv heads][page / 16] groups of
 * 17 * d bytes, d the head size (64, 128 or 256): 16 tokens of one head, as
 *   key codes    [16 tokens][d / 2]
 *   value codes  [d / 128 planes, 1 at d = 64][4][16 runs][4][4 bytes, 2 at d = 64]: token 4 g + i,
 *                run r is 8 consecutive channels (4 at d = 64) of the plane's 128 (64)
 *   key scales   [16 tokens][d / 32]
 *   value scales [d / 32][16 tokens]
 * Codes are e2m1, the low nibble the even channel; a scale byte E is 2^(E - 127) for 32 consecutive
 * channels of one token, 255 for a block that held a value that is not finite. A byte above 252 reads
 * as NaN, whoever wrote it.
 * E is the smallest exponent with amax <= 7 * 2^(E - 127), within 1 .. 252, so that rounding to the
 * nearest code is off by at most 2^(E - 127) at the top; codes round to nearest, ties to even. The
 * value layout puts 4 tokens of a run side by side: a lane of the attention kernels holds the codes
 * that one matrix instruction contracts over as 16 consecutive bytes.
 */
#ifndef KV4_ATTN_H_
#define KV4_ATTN_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KV4_ABI_VERSION 1

enum {
  KV4_OK = 0,
  KV4_EINVAL = 1, /* bad shape, pointer, stride, alignment or page list */
  KV4_EHIP = 3    /* the HIP runtime reported an error at launch */
};

/* Bits of the `flags` arguments. */
enum {
  KV4_PLUS_ONE = 1,   /* the norm's weight is w + 1 (Gemma's convention) */
  KV4_ADJACENT = 2,   /* rotate channels (2p, 2p + 1) instead of (p, p + rot / 2) */
  KV4_TABLE_BF16 = 4, /* cos_sin is bf16 instead of fp32 */
  KV4_POS_I32 = 8,    /* positions are int32 instead of int64 */
  KV4_CAUSAL = 16     /* attention: a query sees no token behind its own place */
};

/* ABI version of the loaded library (KV4_ABI_VERSION). */
int kv4_abi_version(void);

/* Description of the last failure on the calling thread ("" if none). */
const char* kv4_last_error(void);

/* Bytes of one page: heads * page / 16 * 17 * d. */
int kv4_page_bytes(int heads, int page, int d, size_t* bytes);

/* Per-head RMSNorm of q and k and the rotation, one pass:
 *   y = x * (1 / sqrt(mean(x^2) + eps)) * (w [+ 1]),  then channel pairs rotated by their angles,
 * in fp32 with every step fixed (sum of squares: 8 consecutive channels by halves, then the groups
 * of 8 by halves; no fused multiply-add; correctly rounded square root and quotient), rounded to
 * bf16 once. q bf16 [T, q_heads, d] and k bf16 [T, kv_heads, d] with token and head strides in
 * elements (multiples of 8) and 16-byte aligned; q_out, k_out contiguous. A null weight leaves the
 * norm of that tensor out. cos_sin [table_rows][rot]: rot / 2 cosines, then the sines; rot a
 * multiple of 16 up to d, channels from rot on are not rotated (rot 0: none, cos_sin and positions
 * unused). positions [axes][T], row stride pos_stride; pair p turns by the angle at the position
 * on axis axis_of_pair[p] (int32 [rot / 2]; null where axes is 1). A position outside the table or
 * an axis outside 0 .. axes - 1 makes the pair NaN. */
int kv4_qk_norm_rope(const void* q, long q_ts, long q_hs, const void* k, long k_ts, long k_hs,
                     const void* q_weight, const void* k_weight, const void* cos_sin,
                     long table_rows, int rot, const void* positions, long pos_stride, int axes,
                     const int* axis_of_pair, void* q_out, void* k_out, int T, int q_heads,
                     int kv_heads, int d, float eps, int flags, void* stream);

/* kv4_qk_norm_rope with the new keys (rounded from fp32) and values bf16 [T, kv_heads, d] written
 * to the cache instead of a k_out: token t goes to slot slots[t] = page number * page + place (int64
 * [T]; a slot below 0 or past the last page is skipped, slots are distinct). page_stride: bytes from
 * one page to the next, a multiple of 16 below 2^32. */
int kv4_qk_norm_rope_append(const void* q, long q_ts, long q_hs, const void* k, long k_ts,
                            long k_hs, const void* v, long v_ts, long v_hs, const void* q_weight,
                            const void* k_weight, const void* cos_sin, long table_rows, int rot,
                            const void* positions, long pos_stride, int axes,
                            const int* axis_of_pair, void* q_out, void* cache, long pages,
                            long page_stride, int page, const int64_t* slots, int T, int q_heads,
                            int kv_heads, int d, float eps, int flags, void* stream);

/* Tokens of the cache as bf16 k, v [T, heads, d] (exact: e2m1 times a power of two). A slot below 0
 * gives zeros, one past the last page NaN. */
int kv4_gather(const void* cache, long pages, long page_stride, int page, const int64_t* slots,
               void* k, void* v, int T, int heads, int d, void* stream);

/* Softmax attention of the last tokens of `batch` sequences over their cached tokens:
 *   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
 * q bf16 [total, q_heads, d] (token and head strides in elements, multiples of 8; 16-byte aligned),
 * sequence b's queries are rows q_starts[b] .. q_starts[b + 1] - 1 (int32 [batch + 1], at most max_q
 * apart, ascending: with starts that go back, outputs are unspecified) and stand at the end of its
 * seq_lens[b] cached tokens (int32 [batch], at most max_len): query i of n at place p = seq_len - n + i.
 * It sees the tokens j < seq_len, with KV4_CAUSAL j <= p, and with window > 0 j > p - window. A query
 * that sees nothing gives zeros.
 * What a masked token holds, NaN included, has no effect. page_table int32 [batch][table_cols]
 * with row stride table_stride: the sequence's pages in order; entries past its last page are not
 * read. A page number outside the cache makes the outputs of the queries that would read it NaN; a
 * sequence longer than the table's row or max_len, of more queries than max_q, or with tokens in a
 * cache of no pages, all of its. Query head h reads kv head h / (q_heads / kv_heads).
 * out bf16 [total, q_heads, d], contiguous. scale > 0. Scores, softmax statistics and sums are fp32;
 * the weights of the values are rounded to bf16 for the matrix cores. They are relative to a running
 * maximum that may lag by 2^8, so that sums over values beyond 2^100 may pass fp32's range.
 * workspace: kv4_attention_workspace() bytes, 16-byte aligned (may be null for 0), free again when
 * the launches have run. */
int kv4_attention(const void* q, long q_ts, long q_hs, const void* cache, long pages,
                  long page_stride, int page, const int* page_table, long table_stride,
                  int table_cols, const int* seq_lens, const int* q_starts, void* out,
                  void* workspace, size_t workspace_bytes, int total, int batch, int max_q,
                  int max_len, int q_heads, int kv_heads, int d, float scale, int window,
                  int flags, void* stream);

/* Bytes of workspace kv4_attention needs for these sizes (the partial results of long contexts
 * split over workgroups). */
int kv4_attention_workspace(int total, int batch, int max_q, int max_len, int q_heads, int kv_heads,
                            int d, int window, size_t* bytes);

/* Copies page src to page dst for each of the n pairs (int32 [n][2] = src, dst, in HOST memory, read
 * before the call returns) in `layers` caches layer_stride bytes apart, and where tables is not null
 * replaces src by dst in the int32 [table_rows][table_cols] page table (row stride table_stride), in
 * one launch per 448 pairs. No page is both read and written and none written twice; with a table
 * none is read twice either (refused otherwise). */
int kv4_move_pages(void* cache, int layers, long layer_stride, long pages, long page_stride,
                   size_t page_bytes, const int* pairs, int n, int* tables, int table_rows,
                   int table_cols, long table_stride, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KV4_ATTN_H_ */
