/*
 * bi.h -- C ABI of libbi.so, the MI355X (gfx950) batch-invariant GEMM and
 * attention kernels.
 *
 * The reference launches its two Metal kernels through MLX's
 * `mx.fast.metal_kernel` callables; each entry point below replaces exactly one
 * of those launches (cited per function). Plain C types only: no torch, no C++
 * types, no exceptions and no allocation cross this boundary. The caller owns
 * every buffer (device pointers), allocates the output, and passes the HIP
 * stream to launch on (NULL = the default stream). Every call is asynchronous
 * on that stream and safe to record into a HIP graph: the launch path makes no
 * allocation, no host synchronisation and no choice other than the grid that
 * depends on the shape.
 *
 * Every function returns BI_OK (0) or a negative status; bi_last_error() then
 * returns a thread-local message describing the failure. Arguments are
 * validated before any HIP call is made, so argument errors are reported the
 * same way on a machine without a GPU.
 */
#ifndef BI_H
#define BI_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BI_ABI_VERSION 1

/* Element types; the compute is always fp32 accumulate. */
enum bi_dtype { BI_F32 = 0, BI_F16 = 1, BI_BF16 = 2 };

enum bi_status {
  BI_OK = 0,
  BI_EINVAL = -1,       /* bad argument: null pointer, negative size, bad mode, a launch past 2^32 threads */
  BI_EUNSUPPORTED = -2, /* valid but not built: e.g. an attention head dim */
  BI_ELAUNCH = -3       /* the HIP launch itself failed */
};

/* Attention masks (reference _attention.py:173-202, MASK_MODE at :92-97). */
enum bi_mask_mode {
  BI_MASK_NONE = 0,
  BI_MASK_CAUSAL = 1, /* key i is used by query row s iff i <= s + causal_offset */
  BI_MASK_ARRAY = 2   /* additive mask in the element type; <= -3e38 skips the key */
};

/* ABI revision of the loaded library (BI_ABI_VERSION at build time). */
int bi_abi_version(void);

/* Thread-local message for the most recent non-zero return on this thread. */
const char* bi_last_error(void);

/*
 * out[m, n] = T( bias ? alpha * acc + beta * bias[n] : acc ),
 * acc = sum_k a[m, k] * B[k, n] accumulated in fp32.
 *
 * Replaces the bi_gemm launch `_KERNEL(inputs=[a2, b, bias_arr, coef], ...)`
 * at reference mlx_batch_invariant/_gemm.py:212-221 (kernel body
 * _gemm.py:29-130, B load :152-157, grid :210).
 *
 *   a     (M, K) row-major, element type `dtype`
 *   b     trans_b == 0: (K, N) row-major  (bi.matmul / bi.addmm layout)
 *         trans_b == 1: (N, K) row-major  (bi.linear / nn.Linear layout)
 *   bias  (N,) or NULL; alpha and beta are used only when bias is non-NULL
 *   out   (M, N) row-major
 *
 * One workgroup owns the whole K reduction of its output tile. The per-element
 * arithmetic (MFMA instruction, K-chunk order, epilogue) is fixed at compile
 * time and does not depend on M, N, the batch neighbours of a row, its position
 * inside a tile, or whether the call was captured in a graph. M == 0 or
 * N == 0 is a no-op. K == 0 yields the epilogue applied to a zero accumulator.
 */
int bi_gemm(const void* a, const void* b, const void* bias, void* out,
            int64_t M, int64_t N, int64_t K, int dtype, int trans_b,
            float alpha, float beta, void* hip_stream);

/*
 * Single-pass scaled dot product attention; one workgroup owns the whole key
 * reduction of a query row (for the query heads of one kv head together).
 *
 * Replaces the bi_sdpa launch `_KERNEL(inputs=[q, k, v, m, mstride, scale,
 * sinks], ...)` at reference mlx_batch_invariant/_attention.py:241-250 (kernel
 * body _attention.py:32-149).
 *
 *   q     (B, H, qL, D)      element strides qkv_strides[0..2] for (b, h, s)
 *   k     (B, Hkv, N, D)     strides qkv_strides[3..5] for (b, h, n)
 *   v     (B, Hkv, N, V)     strides qkv_strides[6..8] for (b, h, n)
 *         the last dimension of q, k and v is contiguous; qkv_strides == NULL
 *         means all three are fully contiguous
 *   mask  BI_MASK_ARRAY only: element type `dtype`, last dim (N) contiguous,
 *         element strides mask_strides[0..2] for (b, h, s); 0 broadcasts
 *   sinks (H,) logits in `dtype` or NULL (an extra denominator term per head)
 *   out   (B, H, qL, V) contiguous
 *   scale multiplies q.k; H must be a multiple of Hkv (GQA: head h reads
 *         kv head h / (H / Hkv))
 *
 * One fixed reduction per element type. BI_F32: key i is owned by partial
 * (i mod 32) and walked in ascending order; the 32 partials are combined in a
 * fixed order. BI_F16 / BI_BF16 (matrix cores): keys are taken in blocks of
 * 32, block b owned by chain (b mod 4) and walked in ascending order; the 4
 * chains are combined in a fixed order. Nothing in the reduction depends on
 * B, qL, the other query rows, or N beyond which keys exist, so growing the
 * context with masked keys leaves earlier results bitwise unchanged. A query
 * row whose keys are all masked yields 0. A sink enters the fixed-order
 * combine as one more partial (m = sink, l = 1, o = 0).
 * Keys that no query row can see -- past every row's causal bound (e.g. an
 * unwritten cache tail) or hidden by an array mask from every query sharing a
 * workgroup -- never reach the output, whatever they hold (the reference skips
 * them, _attention.py:92-98). The matrix-core path multiplies the values of a
 * key that is visible to another query row of the same 32-key block, but not
 * to this one, by zero; a NaN or infinity there, which reaches that other
 * row's output in any case, may also reach this row's, as an all-NaN row,
 * depending on the launch shape and on which rows share its workgroup. Bit
 * parity across launch shapes, batch sizes and query lengths therefore holds
 * for finite values of every key that some query row of the call can see.
 * Supported head dims (D, V): D == V in {32, 64, 96, ..., 512} (every multiple
 * of 32 up to 512) and (192, 128), (128, 64), (64, 128), (256, 128), (128, 256),
 * (576, 512); other multiples of 32 return BI_EUNSUPPORTED (each pair is a
 * compiled kernel set). fp32 heads above 352 keep part of their state in
 * scratch memory (correct, slower).
 */
int bi_sdpa(const void* q, const void* k, const void* v,
            const void* mask, const int64_t* mask_strides,
            const void* sinks, void* out,
            int64_t B, int64_t H, int64_t Hkv, int64_t qL, int64_t N,
            int64_t D, int64_t V,
            const int64_t* qkv_strides,
            float scale, int mask_mode, int64_t causal_offset,
            int dtype, void* hip_stream);

/*
 * Bytes of device memory with which bi_sdpa_ws is expected to run this problem
 * faster than bi_sdpa; 0 if it would not use any. The current device's compute
 * units decide, and at most 256 MiB are asked for.
 */
int64_t bi_sdpa_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t qL, int64_t N,
                          int64_t D, int64_t V, int dtype, int mask_mode);

/*
 * bi_sdpa, the same bits, with `workspace_bytes` bytes of device memory (at
 * least bi_sdpa_workspace's, 16-byte aligned; with less, or NULL, it is
 * bi_sdpa). A first kernel then writes the raw scores there, its workgroups
 * sharing out the keys, and bi_sdpa's reduction reads them. The call overwrites
 * the memory; it must stay allocated, and unused by others, until the call's
 * work on the stream has run.
 */
int bi_sdpa_ws(const void* q, const void* k, const void* v,
               const void* mask, const int64_t* mask_strides,
               const void* sinks, void* out,
               int64_t B, int64_t H, int64_t Hkv, int64_t qL, int64_t N,
               int64_t D, int64_t V,
               const int64_t* qkv_strides,
               float scale, int mask_mode, int64_t causal_offset,
               int dtype, void* workspace, int64_t workspace_bytes, void* hip_stream);

/*
 * out = x @ dequantize(w).T for an affine-quantized weight, without
 * materialising the dequantized matrix.
 *
 * Replaces the bi_qgemm launch `_QKERNEL(inputs=[x, w, scales, qbias, ...])`
 * at reference mlx_batch_invariant/_gemm.py:275-284 (quantized_linear
 * :243-285; the kernel's dequantizing B load :163-177).
 *
 *   x       (M, K) row-major, dtype BI_F16 or BI_BF16, 16-byte aligned
 *   w       (N, K * bits / 32) uint32, 16-byte aligned: weight element k of
 *           row n is bits bits * (k % (32 / bits)) .. of word k / (32 / bits)
 *           of that row (little-endian packing, the MLX affine layout)
 *   scales, (N, K / group_size) in the element type of x; element k of row n
 *   biases  dequantizes to the fp32 value
 *           v = fp32(scales[n][k/group] * q + biases[n][k/group])
 *   out     (M, N) row-major
 *   bits in {2, 4, 8}; group_size in {32, 64, 128} and dividing K.
 *
 * As in the reference kernel (a float B tile, _gemm.py:46, :170-173), v is
 * not rounded to the element type. The product is formed per group in fp32:
 * P = sum x_k * q_k and X = sum x_k over the group's 32-element chunks of K
 * (MFMAs with exact products), then acc = fma(scale, P, acc) and
 * acc = fma(bias, X, acc), groups in ascending order; the output is rounded
 * once. This is sum_k x_k * v_k with fp32 roundings only, the same sequence
 * for every output element: nothing depends on M or on a row's batch
 * neighbours. BI_F32 activations return BI_EUNSUPPORTED.
 */
int bi_qgemm(const void* x, const void* w, const void* scales, const void* biases, void* out,
             int64_t M, int64_t N, int64_t K, int group_size, int bits, int dtype,
             void* hip_stream);

/*
 * Block tables and slot maps of a serving step over a paged cache, from the
 * requests' lengths. Request r holds context_lens[r] rows and brings
 * new_lens[r] more (negative lengths count as 0); its row i is row
 * i % page_size of page block_tables[r][i / page_size].
 *
 *   block_tables (R, W) int32, rows table_stride apart, updated in place: the
 *                pages that the new rows begin are taken from free_pages in
 *                the requests' order, from its front; -1 where the F free
 *                pages do not reach. No other entry is written. Rows past
 *                W * page_size have no page.
 *   slots        (T) page * page_size + row of every new token, -1 for one
 *                without a page (or one so far out that this passes 31 bits)
 *                and behind the last token
 *   positions    (T) its row in the request, -1 behind the last token
 *   query_start  (R + 1) first token of every request, and their number
 *   seq_lens     (R) context_lens + new_lens
 *   pages_used   (1) pages the new rows begin (more than F: not all were there)
 *
 * Where the new tokens are more than T, the first T have their slots written
 * and all their pages; the sums must stay below 2^31.
 */
int bi_page_tables(int32_t* block_tables, const int32_t* context_lens, const int32_t* new_lens,
                   const int32_t* free_pages, int32_t* slots, int32_t* positions,
                   int32_t* query_start, int32_t* seq_lens, int32_t* pages_used,
                   int64_t R, int64_t W, int64_t table_stride, int64_t F, int64_t T,
                   int64_t page_size, void* hip_stream);

/*
 * Writes T tokens' keys and values into a paged cache: row slots[t] %
 * page_size of page slots[t] / page_size takes k[t] and v[t]; a slot that is
 * negative or not below num_pages * page_size writes nothing. Slots are
 * distinct (of two tokens with one slot either may be kept, unit by unit).
 *
 *   k (T, Hkv, D), v (T, Hkv, V)     element strides strides[0..1], [2..3]
 *   k_cache (num_pages, Hkv, page_size, D)   strides[4..6] (page, head, row)
 *   v_cache (num_pages, Hkv, page_size, V)   strides[7..9]
 *   the last dimension of each is contiguous
 */
int bi_paged_update(const void* k, const void* v, void* k_cache, void* v_cache,
                    const int32_t* slots, int64_t T, int64_t Hkv, int64_t D, int64_t V,
                    int64_t num_pages, int64_t page_size, const int64_t* strides, int dtype,
                    void* hip_stream);

/*
 * Causal attention of new tokens over a paged cache that already holds their
 * keys and values (bi_paged_update). Tokens query_start[r] ..
 * query_start[r + 1] - 1 are the last ones of request r's seq_lens[r] rows:
 * the last token sees every row, the one before it all but one. With window >
 * 0 a token at position p sees rows j with p - window < j <= p, and the first
 * sink_tokens rows (j < sink_tokens, j <= p); window 0 is none.
 *
 *   q            (T, H, D)    strides[0..1] (token, head)
 *   k_cache      (num_pages, Hkv, page_size, D)  strides[2..4] (page, head, row)
 *   v_cache      (num_pages, Hkv, page_size, V)  strides[5..7]
 *                pointers and strides are multiples of 16 bytes
 *   block_tables (R, W) int32, rows strides[8] apart. A row whose entry is not
 *                a page of the cache, or lies past the table, is not seen.
 *   query_start  (R + 1), seq_lens (R) int32
 *   sinks        (H,) logits in `dtype`, or NULL: one more term of each
 *                head's denominator
 *   out          (T, H, V) contiguous; a token that no request owns, and one
 *                that sees nothing, is 0
 *   max_query, max_seq   bounds of the requests' new tokens and lengths that
 *                the launch may rely on; a request beyond one of them gets NaN
 *   workspace    at least bi_paged_attention_workspace bytes, 16-byte aligned,
 *                or NULL: slower, with the same bits
 *
 * Arithmetic (bi_paged_attn_kernel.h): keys are taken by their position in the
 * request, in segments of a fixed length whose results are folded in order,
 * so that a token's bits depend on its own request's rows alone: not on other
 * requests, on how many tokens are new, on the pages, on the workspace or on
 * rows it does not see. bi_window_attention gives the same bits for the same
 * rows in contiguous memory. (Not bi_sdpa's bits: its chains have no segments.)
 * Rows that a token does not see never reach its output, whatever they hold:
 * not a NaN or infinity either that another token of its request sees. (Calls
 * of many tokens per request that meet one in such a row of values take up to a
 * hundred times as long.)
 * Built for (D, V) in {(64, 64), (96, 96), (128, 128), (192, 128), (192, 192),
 * (256, 256)}.
 */
int bi_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                       const int32_t* block_tables, const int32_t* query_start,
                       const int32_t* seq_lens, const void* sinks, void* out, int64_t T, int64_t R,
                       int64_t H, int64_t Hkv, int64_t D, int64_t V, int64_t num_pages,
                       int64_t page_size, int64_t W, const int64_t* strides, float scale,
                       int64_t window, int64_t sink_tokens, int64_t max_query, int64_t max_seq,
                       int dtype, void* workspace, int64_t workspace_bytes, void* hip_stream);

/* Bytes with which bi_paged_attention runs fastest; 0 if it would use none. */
int64_t bi_paged_attention_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D,
                                     int64_t V, int64_t window, int64_t sink_tokens,
                                     int64_t max_query, int64_t max_seq, int dtype);

/*
 * Causal attention with a sliding window and first tokens that stay visible,
 * over contiguous keys: the rule, types, head dims and bits of
 * bi_paged_attention for B requests of N rows each, the last qL of them new.
 *
 *   q (B, H, qL, D), k (B, Hkv, N, D), v (B, Hkv, N, V): element strides
 *   strides[0..2], [3..5], [6..8] for all but the contiguous last dimension;
 *   out (B, H, qL, V) contiguous. qL may be more than N: the first rows then
 *   see nothing and are 0.
 */
int bi_window_attention(const void* q, const void* k, const void* v, const void* sinks, void* out,
                        int64_t B, int64_t H, int64_t Hkv, int64_t qL, int64_t N, int64_t D,
                        int64_t V, const int64_t* strides, float scale, int64_t window,
                        int64_t sink_tokens, int dtype, void* workspace, int64_t workspace_bytes,
                        void* hip_stream);

/* Bytes with which bi_window_attention runs fastest; 0 if it would use none. */
int64_t bi_window_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t qL, int64_t N,
                                      int64_t D, int64_t V, int64_t window, int64_t sink_tokens,
                                      int dtype);

/*
 * bi_paged_update for a cache of 8 bits: a row of one token and head is kept as
 * whole numbers c in -127 .. 127 and a scale s, its values being c * s.
 *
 *   k_cache, v_cache    int8, strides[4..9] as in bi_paged_update
 *   k_scales, v_scales  (num_pages, Hkv, page_size) float, element strides
 *                       scale_strides[0..2] and [3..5] (page, head, row)
 *   keep_scales 0       s = max |x| / 127 is written for every token and head,
 *                       and c = x / s rounded to the nearest, ties to even. A
 *                       row of zeros has s = 0; one with an infinity or NaN
 *                       s = NaN and codes 0, so that it reads as NaN.
 *   keep_scales 1       the scales are read (not negative; they may lie at
 *                       strides of 0, one for a page or a head); what passes
 *                       127 s is cut off, a NaN is 0, as all is where s = 0
 *
 * Codes and scale depend on the row alone.
 */
int bi_paged_update_q8(const void* k, const void* v, int8_t* k_cache, int8_t* v_cache,
                       float* k_scales, float* v_scales, const int32_t* slots, int64_t T,
                       int64_t Hkv, int64_t D, int64_t V, int64_t num_pages, int64_t page_size,
                       const int64_t* strides, const int64_t* scale_strides, int keep_scales,
                       int dtype, void* hip_stream);

/*
 * The way back: rows of a paged cache as tokens. k[t] (T, Hkv, D) and v[t] (T,
 * Hkv, V) become row slots[t] % page_size of page slots[t] / page_size, zeros
 * where the slot is negative or not below num_pages * page_size. With scales the
 * cache is int8 and a value is c * s in 32 bits, rounded once to `dtype`; with
 * NULL for both it is of `dtype` and copied. Strides as in bi_paged_update_q8.
 */
int bi_paged_read(const void* k_cache, const void* v_cache, const float* k_scales,
                  const float* v_scales, const int32_t* slots, void* k, void* v, int64_t T,
                  int64_t Hkv, int64_t D, int64_t V, int64_t num_pages, int64_t page_size,
                  const int64_t* strides, const int64_t* scale_strides, int dtype,
                  void* hip_stream);

/*
 * bi_paged_attention over a cache of 8 bits: the same rule, with keys k_cache *
 * k_scales and values v_cache * v_scales.
 *
 *   k_cache, v_cache    int8, strides[2..7] as in bi_paged_attention (pointers
 *                       and strides are multiples of 16 bytes)
 *   k_scales, v_scales  (num_pages, Hkv, page_size) float, element strides
 *                       scale_strides[0..2] and [3..5] (page, head, row; 0 for
 *                       one a page or a head)
 *   dtype               of q, sinks and out: BI_F16 or BI_BF16
 *
 * Pages and rows (strides[2], [4], [5], [7] and those of the scales) lie less
 * than 4 GiB apart, none at a negative stride (else BI_EUNSUPPORTED); heads at any
 * stride, and all at any offset.
 *
 * Scores are sums of exact products of codes and q in 32 bits times the row's
 * scale in 32 bits; weights times the row's scale are rounded to `dtype` (BI_F16:
 * but for the scale's power of two, which goes with the codes, so that scales from
 * 2^-14 lose nothing; those of 2^19 and above, of values past 6e7, overflow, and
 * beside scores past 2^26 those of 2^13), products and sums are of 32 bits, the
 * denominator the sum of the weights of 32 bits. A token that sees a row whose key
 * or value scale is infinite or NaN, or whose key scale is negative, is NaN, and so
 * is one whose largest score times log2 e is 2^30 (BI_F16: 2^28) or more from 0
 * within some 512 rows; a score below the range of 32 bits is -inf, and its row not
 * seen. A token's bits depend on its own request's rows alone, as there, and nothing
 * in a row that a token does not see reaches it.
 */
int bi_paged_attention_q8(const void* q, const int8_t* k_cache, const int8_t* v_cache,
                          const float* k_scales, const float* v_scales,
                          const int32_t* block_tables, const int32_t* query_start,
                          const int32_t* seq_lens, const void* sinks, void* out, int64_t T,
                          int64_t R, int64_t H, int64_t Hkv, int64_t D, int64_t V,
                          int64_t num_pages, int64_t page_size, int64_t W, const int64_t* strides,
                          const int64_t* scale_strides, float scale, int64_t window,
                          int64_t sink_tokens, int64_t max_query, int64_t max_seq, int dtype,
                          void* workspace, int64_t workspace_bytes, void* hip_stream);

/* Bytes with which bi_paged_attention_q8 runs fastest; 0 if it would use none. */
int64_t bi_paged_attention_q8_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D,
                                        int64_t V, int64_t window, int64_t sink_tokens,
                                        int64_t max_query, int64_t max_seq, int dtype);

/* Of these, the bytes without which single tokens are computed as slowly as chunks
 * (the rest holds rows laid out); 0 if there are none. */
int64_t bi_paged_attention_q8_least_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                              int64_t D, int64_t V, int64_t window,
                                              int64_t sink_tokens, int64_t max_query,
                                              int64_t max_seq, int dtype);

/*
 * Rotary positions: pair i of every head of token t turns by the angle
 * positions[t] * inv_freq[i], (x, y) -> scale * (x cos - y sin, x sin + y cos).
 *
 *   q (T, H, D), k (T, Hkv, D)   element strides strides[0..1], [2..3] (token,
 *                head), the last dimension contiguous; H or Hkv may be 0
 *   q_out, k_out contiguous, not overlapping q and k
 *   positions    (T) int32, of either sign
 *   inv_freq     (n) doubles, radians per position
 *   interleaved  0: pair i is dims offset + i and offset + n + i;
 *                1: dims offset + 2 i and offset + 2 i + 1
 * The other dims are copied. Angles are reduced in 64 bits; a token's result
 * depends on the token alone.
 */
int bi_rotary(const void* q, const void* k, void* q_out, void* k_out, const int32_t* positions,
              const double* inv_freq, int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t n,
              int64_t offset, const int64_t* strides, float scale, int interleaved, int dtype,
              void* hip_stream);

/*
 * Log probabilities of given tokens under rows of logits, the rows' entropies,
 * and their `top` largest logits.
 *
 *   logits       (rows, V), rows `stride` elements apart
 *   tokens       (rows) of token_bytes 4 or 8; one that is not in 0 .. V - 1
 *                has the log probability NaN
 *   logprobs     (rows) ln softmax(logits)[token]
 *   entropy      (rows) -sum p ln p, in nats; -inf logits count for nothing
 *   top_ids, top_logprobs  (rows, top) in descending order, ties by ascending
 *                id; top is at most 64 and at most V. A NaN logit counts as the
 *                largest.
 * Log probabilities and entropy of a row with a NaN or +inf, or of -inf alone,
 * are NaN. A row's results depend on the row alone.
 */
int bi_token_logprobs(const void* logits, const void* tokens, float* logprobs, float* entropy,
                      int64_t* top_ids, float* top_logprobs, int64_t rows, int64_t V,
                      int64_t stride, int64_t top, int token_bytes, int dtype, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* BI_H */
