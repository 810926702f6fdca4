/*
 * rxq4.h -- C ABI of the MI355X (gfx950) Q4_K weight-path library.
 *
 * Plain C: pointers, sizes and int status codes, no C++ or torch types.  The
 * first seven entry points replace, one for one, the kernel-layer functions
 * that reflex-infer's dispatcher binds (reference
 * src/kernels/kernel_entrypoints.h:7-13, defined in src/kernels/q4_gemm.cu);
 * the C++ API of include/reflex/infer.h is implemented on top of them.  The
 * entry points marked NEW have no reference counterpart: they expose work
 * the reference API cannot express (bf16 GEMM, batched embedding gather,
 * small-batch decode, the quantiser used to build inputs, and the operators
 * of a serving step between the projections: head norms, rotation and the
 * store in a paged cache, attention over it, the next token's draw).
 *
 * Conventions for every entry point:
 *   - `w` is a DEVICE pointer to raw GGML blocks of `ggml_type`: Q4_K (12,
 *     144 bytes per 256 weights), Q5_K (13, 176 bytes) or Q6_K (14, 210
 *     bytes); rows of K/256 blocks, row-major, the base 16-byte aligned.
 *     The embedding entry points take Q4_K and Q6_K, as the reference.
 *     Pointer resolution of host/mmap pointers happens above this layer
 *     (rxq4_resolve_weights).
 *   - fp16/bf16 buffers are raw 16-bit patterns; x must be 16-byte aligned.
 *   - K must be a positive multiple of 256 and at most RXQ4_MAX_K.
 *   - `stream` is a hipStream_t (NULL = null stream).  Calls only enqueue
 *     work; no entry point but rxq4_release_workspace synchronises the
 *     device or the stream.  The one allocation is the fp32 workspace of the
 *     split launches (split-K GEMM with few output tiles, small-batch
 *     products on long rows, attention over long cached contexts), of
 *     rxq4_sample_f32's bins and rxq4_select_pages' scores: 48 MiB
 *     per (device, stream), made by the first such launch on that stream,
 *     never resized, and kept until rxq4_release_workspace(stream) frees it,
 *     so a HIP graph captured on a stream stays valid whatever runs later,
 *     and launches on different streams never share it.  hipStreamPerThread
 *     names a different stream in every thread, so its workspace is kept per
 *     (device, thread).  That first allocation is also legal while the
 *     stream is being captured.
 *   - x must be 16-byte aligned (the one alignment rule the reference does
 *     not have).  Weight blocks need the alignment of their format: Q4_K
 *     and Q5_K 16 bytes, Q6_K 2 bytes (its 210-byte blocks; a row slice of a
 *     Q6_K tensor is accepted wherever it starts).
 *   - The return value is a reflex::infer::Status value (RXQ4_STATUS_*).
 *     On an error nothing is launched; rxq4_last_error() says why.
 */
#ifndef RXQ4_H
#define RXQ4_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Values of reflex::infer::Status (reference include/reflex/infer.h:16-23). */
#define RXQ4_STATUS_SUCCESS 0
#define RXQ4_STATUS_UNSUPPORTED_DEVICE 1
#define RXQ4_STATUS_UNSUPPORTED_MODEL 2
#define RXQ4_STATUS_UNSUPPORTED_QUANT_FORMAT 3
#define RXQ4_STATUS_INVALID_ARGUMENT 4
#define RXQ4_STATUS_NOT_IMPLEMENTED 5

#define RXQ4_GGML_TYPE_Q4_K 12
#define RXQ4_GGML_TYPE_Q5_K 13
#define RXQ4_GGML_TYPE_Q6_K 14
#define RXQ4_MAX_K 65536
/* Limits of the serving entry points (rxq4_qk_norm_rope and _axes, rxq4_attention_paged_f16,
 * rxq4_kv_bounds, rxq4_select_pages, rxq4_attention_selected_f16, rxq4_sample_f32, whose
 * n_rows is at most RXQ4_MAX_TOKENS). */
#define RXQ4_MAX_SEQS 65536
#define RXQ4_MAX_TOKENS 1048576
#define RXQ4_MAX_POSITIONS 16777216
#define RXQ4_MAX_HEADS 1024
#define RXQ4_MAX_VOCAB 4194304
#define RXQ4_MAX_AXES 16
#define RXQ4_MAX_SELECT 4096

/* Element types for the typed GEMM entry point. */
#define RXQ4_DTYPE_F32 0
#define RXQ4_DTYPE_F16 1
#define RXQ4_DTYPE_BF16 2

/* One output range of a multi-matrix GEMV sharing one x (pair = 2, triple = 3). */
typedef struct rxq4_rows {
    void *y;           /* fp16 [M] */
    const void *w;     /* device blocks of ggml_type [M x K/256] */
    int ggml_type;
    int M;
} rxq4_rows;

/* y[M] fp16 = RNE(W[M x K] . x[K]), fp32 accumulation.
 * Replaces kernels::gemv_quant (reference q4_gemm.cu:2031-2036, 1856-1914). */
int rxq4_gemv_f16(void *y, const void *w, int ggml_type, const void *x, int M, int K,
                  void *stream);

/* y[M] fp16 = RNE(float(RNE(W . x)) + float(residual)); y may equal residual.
 * Replaces kernels::gemv_quant_add (reference q4_gemm.cu:2038-2045, 755-779). */
int rxq4_gemv_add_f16(void *y, const void *w, int ggml_type, const void *x,
                      const void *residual, int M, int K, void *stream);

/* 1..3 independent GEMVs sharing x, one launch (ranges may mix Q4_K, Q5_K
 * and Q6_K).
 * Replaces kernels::gemv_quant_pair (reference q4_gemm.cu:2047-2056) with
 * n_ranges = 2 and kernels::gemv_quant_triple (q4_gemm.cu:2058-2069) with 3. */
int rxq4_gemv_multi_f16(const rxq4_rows *ranges, int n_ranges, const void *x, int K,
                        void *stream);

/* y[M] fp32 = W . x (logits).
 * Replaces kernels::gemv_quant_f32 (reference q4_gemm.cu:2071-2076, 491-507). */
int rxq4_gemv_f32(float *y, const void *w, int ggml_type, const void *x, int M, int K,
                  void *stream);

/* y[N x M] fp16 (token-major) = x[N x K] fp16 . W^T.  N == 1 is the GEMV;
 * for Q4_K, N <= 4 runs the decode GEMV with every token's activations in
 * registers (per token bit-identical to the GEMV), N <= 16 the multi-token
 * MFMA kernel, larger N the MFMA GEMM; Q5_K / Q6_K run their multi-token
 * MFMA kernel up to N = 16 (large Q5_K matrices the GEMM) and the same GEMM
 * above.  Small matrices run more than 16 tokens through the multi-token
 * kernels too, in chunks of 16.
 * Replaces kernels::gemm_quant_batched (reference q4_gemm.cu:2023-2029,
 * 1707-1740). */
int rxq4_gemm_f16(void *y, const void *w, int ggml_type, const void *x, int M, int N,
                  int K, void *stream);

/* dst[hidden] fp16 = dequant(W[token_id, :]), bit-exact.
 * Replaces kernels::dequant_embedding_row (reference q4_gemm.cu:2078-2115).
 * Like the reference, token_id is not range-checked (no vocab size given). */
int rxq4_embed_row_f16(void *dst, const void *w, int ggml_type, int token_id,
                       int hidden_dim, void *stream);

/* NEW.  Typed GEMM: y[N x M] (y_dtype) = x[N x K] (x_dtype) . W^T.
 * Supported: x F16 -> y F16|F32, x BF16 -> y BF16|F32.  Weight tiles are
 * dequantised to the x type, products accumulate in fp32. */
int rxq4_gemm(void *y, int y_dtype, const void *w, int ggml_type, const void *x,
              int x_dtype, int M, int N, int K, void *stream);

/* NEW.  rxq4_gemm with no allocation: same arguments, routing, kernels and
 * results, but the fp32 partials of its split launches live in a fixed
 * 48 MiB device array of the library (one per device, made by the HIP
 * runtime when the entry point is first called on that device and held
 * until the process ends) instead of the stream's workspace, so no call ever allocates device
 * memory (no hipMalloc/hipFree/allocating library call).  No counterpart in
 * the reference; it is for callers that cannot allocate: code under HIP graph
 * capture, serving loops, harnesses that forbid allocation.  No shape is
 * refused for the array's size: the launchers shrink their split counts so
 * that the partials fit it (the same counts as rxq4_gemm, whose workspace has
 * the same size, so the results are identical).  The array keeps the last call's
 * contents and every call on a device shares it: calls that overlap on one
 * device (two streams, or two threads) race and must be serialised by the
 * caller. */
int rxq4_gemm_noalloc(void *y, int y_dtype, const void *w, int ggml_type, const void *x,
                      int x_dtype, int M, int N, int K, void *stream);

/* NEW.  Batched gather: dst[i, :] fp16 = dequant(W[ids[i], :]) for i < n_ids.
 * ids is a device int32 array; ids outside [0, n_vocab) give a zero row. */
int rxq4_embed_rows_f16(void *dst, const void *w, int ggml_type, int64_t n_vocab,
                        const int32_t *ids, int n_ids, int hidden_dim, void *stream);

/* NEW.  Quantise fp32 rows [n_rows x K] (device) to Q4_K blocks (device)
 * with a plain per-sub-block min/max fit (fast; not ggml's search). */
int rxq4_quantize_q4k(void *dst, const float *src, int64_t n_rows, int K, void *stream);

/* NEW.  Quantise fp32 rows [n_rows x K] (device, 16-byte aligned) to blocks
 * of ggml_type 12 (Q4_K), 13 (Q5_K) or 14 (Q6_K) (device; 16-byte aligned,
 * Q6_K 2-byte) with ggml's reference quantisers, byte for byte what
 * llama.cpp's quantize_row_q{4,5,6}_K_ref write without an importance
 * matrix (ggml-quants.c), so synthetic weights match real GGUF files
 * statistically.  No reference counterpart: the reference ships no
 * quantiser and reads these formats (q4_gemm.cu:147-171). */
int rxq4_quantize(void *dst, int ggml_type, const float *src, int64_t n_rows, int K,
                  void *stream);

/* out[n_heads x head_dim] fp16 = attention of one query token over KV
 * positions [0, seq_len): per head h (KV head h / (n_heads / n_kv_heads)),
 * softmax(scale * q.K^T) V with fp32 softmax.  k_cache / v_cache are
 * [pos][n_kv_heads][head_dim], fp16, or int8 when kv_int8 != 0 with optional
 * per-(position, KV head) fp32 scales k_scales / v_scales [pos][n_kv_heads]
 * (NULL = 1).  head_dim a multiple of 8 (int8: 16), at most 256; n_heads a
 * multiple of n_kv_heads.  Decode splits long sequences over the stream's
 * workspace described above.
 * Replaces kernels::flash_attention_decode (reference attention.cu:450-466,
 * 41-173). */
int rxq4_attention_decode_f16(void *out, const void *q, const void *k_cache,
                              const void *v_cache, int n_heads, int n_kv_heads, int head_dim,
                              int seq_len, float scale, int kv_int8, const float *k_scales,
                              const float *v_scales, void *stream);

/* Prefill: N query tokens q[N x n_heads x head_dim]; token t attends to
 * positions [0, start_pos + t + 1) of the caches (causal).  What the caches
 * hold past a token's last position does not reach its row, infinities and NaN
 * included, with one exception: at head_dim 64 and 128, where the launcher picks
 * the kernel for short prompts, an infinity or NaN in V or v_scales may reach
 * the earlier tokens of its 64-position tile.  Few tokens on long contexts split
 * over the stream's workspace as decode does (without room for one the launch
 * runs unsplit): a graph captured with such a call uses the capturing stream's,
 * also where it is replayed on another, and must not be replayed once
 * rxq4_release_workspace has freed it.
 * Replaces kernels::flash_attention_prefill_batched (reference
 * attention.cu:432-448, 180-290). */
int rxq4_attention_prefill_f16(void *out, const void *q, const void *k_cache,
                               const void *v_cache, int n_heads, int n_kv_heads, int head_dim,
                               int N, int start_pos, float scale, int kv_int8,
                               const float *k_scales, const float *v_scales, void *stream);

/* NEW.  A paged KV cache of one layer, shared by the sequences of a batch.
 * Page p holds page_size consecutive positions of one sequence as
 * [slot][n_kv_heads][head_dim], page_stride elements after page p - 1 (0: dense;
 * e.g. K and V pages alternating in one allocation have twice the dense
 * stride).  fp16, or int8 with per-(position, KV head) fp32 scales
 * [n_pages][page_size][n_kv_heads] (NULL: 1, for reading only).  Row i of
 * page_table names the pages of sequence i in order; NULL: one sequence whose
 * page j is page j, i.e. a contiguous cache [pos][n_kv_heads][head_dim].  An
 * entry outside [0, n_pages) is a hole: its positions are never read or
 * written, and no token attends to them.  Pages may be shared by sequences as
 * long as no call writes to a shared slot.  page_size: a power of two, 1 to
 * 1024; head_dim and alignment as the attention entry points above; n_pages *
 * page_size below 2^31. */
typedef struct rxq4_paged_kv {
    void *k, *v;
    float *k_scales, *v_scales;
    const int32_t *page_table;   /* device, [n_seqs][table_stride] */
    int64_t page_stride;         /* elements from page to page, 0: dense */
    int table_stride;            /* entries per sequence */
    int n_pages;
    int page_size;
    int n_kv_heads;
    int head_dim;
    int kv_int8;
} rxq4_paged_kv;

/* NEW.  The new tokens of a batch of sequences: those of sequence i are the rows
 * [q_starts[i], q_starts[i + 1]) of q and the like, and the last of its
 * seq_lens[i] positions (its cached positions and the new ones).  Both arrays
 * are in device memory, so a captured launch can be replayed with other
 * lengths as long as the limits below hold.  Rows before q_starts[0] and from
 * q_starts[n_seqs] on (a padded batch) are left as they are.  A token whose
 * position would be negative (seq_lens[i] below the new tokens) attends to
 * nothing. */
typedef struct rxq4_seq_batch {
    const int32_t *q_starts;   /* device, [n_seqs + 1], ascending */
    const int32_t *seq_lens;   /* device, [n_seqs] */
    int n_seqs;
    int n_tokens;   /* rows of q: a limit of every q_starts value */
    int max_new;    /* no sequence has more new tokens (those past it are not computed) */
    int max_len;    /* no seq_lens value is larger (positions past it are not seen) */
} rxq4_seq_batch;

/* NEW.  The step between a layer's Q/K/V projection and its attention, in one
 * pass: RMS norm of every query and key head (q_weight, k_weight: fp32
 * [head_dim], NULL: none), rotation of the first n_rot dims of queries and keys
 * by position * inv_freq[i] (fp32 [n_rot / 2], device; the product in 64 bits)
 * in pairs (i, i + n_rot / 2), or (2 i, 2 i + 1) where `interleaved`, and the
 * store of keys and values into the cache's slots of their positions.
 *   q_out   fp16 [n_tokens][n_heads][head_dim]; may be q itself where that is
 *           fp16 with the same stride, and overlap q, k and v in no other way
 *   q, k, v x_dtype (F16, BF16, F32), 16-byte aligned, rows q_stride / kv_stride
 *           elements apart (multiples of 8): slices of one fused output, or
 *           three arrays
 * Everything is computed in fp32 and rounded once.  int8 caches get scale =
 * max |row| / 127 and rint(row / scale) per position and head, both scale arrays
 * given; a row with a NaN gets a NaN scale, one with an infinity an infinite
 * one (either reads as NaN).  Tokens at negative positions get a zero query
 * row; keys and values whose position is negative, in a hole or past the table
 * are not stored.  Two rows for one slot (a page shared by sequences) race.
 * No counterpart in the reference, whose KernelSupport names rope, rmsnorm and
 * kv_convert and leaves them to its caller. */
int rxq4_qk_norm_rope(void *q_out, const void *q, const void *k, const void *v, int x_dtype,
                      int64_t q_stride, int64_t kv_stride, int n_heads, const float *q_weight,
                      const float *k_weight, float eps, const float *inv_freq, int n_rot,
                      int interleaved, const rxq4_seq_batch *batch, const rxq4_paged_kv *cache,
                      void *stream);

/* NEW.  Attention of each sequence's new tokens over its pages: a token at
 * position p attends to positions [0, p] (causal), holes left out; fp32
 * softmax, fp16 q and out [n_tokens][n_heads][head_dim]; out may be q itself, and
 * overlap it in no other way.  A batch may mix decoding sequences (one new
 * token), drafts and prompt chunks.  A token that sees nothing gets zeros.  What the cache holds at positions a token does not see
 * does not reach its row, infinities and NaN included.  Few tokens on long
 * contexts split over the stream's workspace described above (a graph captured
 * with such a call uses the capturing stream's, also where it is replayed on
 * another).  The split depends on the whole batch: the same batch gives the same
 * bits, a sequence in another batch the same within rounding.
 * What the split follows, rows being new tokens x n_heads / n_kv_heads:
 *   sequences of up to 16 rows   the lengths on the device, in batches of up to 256
 *       sequences; max_len and table_stride may be capacities.  Past 256 the host's
 *       limits: max_len or table_stride far above the lengths leave long chunks
 *   sequences of more            the lengths on the device too, but only where
 *       n_tokens * n_heads is below 128 per CU and the batch has at most 1024
 *       sequences.  Above either no sequence is split: a short chunk after a long
 *       context goes apart from some hundred decoding sequences or padding rows
 * No counterpart in the reference, whose KernelSupport names
 * paged_decode_attention. */
int rxq4_attention_paged_f16(void *out, const void *q, int n_heads, float scale,
                             const rxq4_seq_batch *batch, const rxq4_paged_kv *cache,
                             void *stream);

/* NEW.  rxq4_qk_norm_rope with the angles from coordinates of the caller's instead of
 * the position in the cache: tokens of images and video have a time, a height and a
 * width, and text behind them does not go on at the cache's position.
 *   positions  int32, device: the coordinate of token t (a row of q) on axis a is
 *              positions[a * position_stride + t], any whole number; n_axes axes, 1 to 16.
 *              position_stride: n_tokens or more (2^32 at most), or 0: one row for all axes
 *   axis_of    int32 [n_rot / 2], device: the axis whose coordinate turns pair i, times
 *              inv_freq[i]; a value outside [0, n_axes) counts as coordinate 0.  NULL:
 *              axis 0 for every pair
 * Everything else is rxq4_qk_norm_rope's, the slots of keys and values included: they
 * follow from seq_lens.  With the cache's positions on one axis the results are its, bit
 * for bit.  q_out may not overlap positions or axis_of.
 * No counterpart in the reference (rxq4_qk_norm_rope). */
int rxq4_qk_norm_rope_axes(void *q_out, const void *q, const void *k, const void *v, int x_dtype,
                           int64_t q_stride, int64_t kv_stride, int n_heads, const float *q_weight,
                           const float *k_weight, float eps, const float *inv_freq, int n_rot,
                           int interleaved, const int32_t *positions, int64_t position_stride,
                           int n_axes, const int32_t *axis_of, const rxq4_seq_batch *batch,
                           const rxq4_paged_kv *cache, void *stream);

/* NEW.  Attention over chosen pages, for long contexts, is three calls beside a paged
 * cache: bounds of the pages' keys, kept up as tokens are stored; the choice of each
 * token's pages by a score against the bounds; attention over the chosen pages.
 *
 * rxq4_kv_bounds: for every page that new tokens of the batch went to (rxq4_qk_norm_rope
 * has stored them), and each KV head, the smallest and the largest key of each dim over
 * the page's positions that its sequence has filled, computed anew.
 *   bounds  int8 [n_pages][n_kv_heads][head_dim / 8][2][8], 16-byte aligned: of each 8 dims
 *           the smallest, then the largest, rint(x / scale)
 *   scales  fp32 [n_pages][n_kv_heads]: max(|smallest|, |largest|) * fp32(1 / 127) over
 *           the dims,
 * lying beside the pool as the int8 scales do.  A NaN key is left out (a dim with
 * nothing else gets 0); an infinity counts as fp32's largest number.  Positions and pages
 * that rxq4_qk_norm_rope would not store to are left out.  Two sequences with new tokens
 * in one page race.  A prompt's pages that came with their keys (a prefix that is shared
 * or loaded) get theirs from a call whose batch has all its tokens as new ones; the batch's
 * rows stand for no arrays here. */
int rxq4_kv_bounds(void *bounds, float *scales, const rxq4_seq_batch *batch,
                   const rxq4_paged_kv *cache, void *stream);

/* NEW.  The pages that each new token's queries (fp16 [n_tokens][n_heads][head_dim], 16-byte
 * aligned, after rotation) attend to, for each KV head.
 *   pages    int32 [n_tokens][n_kv_heads][n_select]: places in the sequence's row of
 *            page_table, ascending; -1 behind the last.  n_select: 1 to 4096
 *   chosen   of the pages in the pool with a position that the token sees: the first
 *            n_first and the last n_last of the sequence (holes among them are left out),
 *            and those with the largest scores until there are n_select, of equal scores
 *            the first pages.  n_first + n_last is at most n_select.  (n_last 1 or more
 *            keeps the page that the token itself is in)
 *   score    the largest, over the heads of the KV head's group, of
 *            (sum_d max(z_d lo_d, z_d hi_d)) * step * scale, in this order in fp32, where
 *            lo, hi and scale are the page's bounds, step = max |q| * fp32(1 / 127) and z =
 *            rint(q / step) of the head's query (NaN as 0, infinities as 65504): up to the
 *            steps no key of the page has a larger product with the query.  The sum is
 *            exact, so the lists do not depend on how the work is cut
 * Bounds and scales are rxq4_kv_bounds' (a page whose scale is negative or NaN is not
 * chosen for its score; an infinite one times a sum of 0 is 0).  Tokens that see nothing get -1s.  Rows of no sequence, and of
 * tokens past max_new, are left as they are.  A few tokens with many pages use the
 * stream's workspace described above. */
int rxq4_select_pages(int32_t *pages, int n_select, int n_first, int n_last, const void *q,
                      int n_heads, const void *bounds, const float *scales,
                      const rxq4_seq_batch *batch, const rxq4_paged_kv *cache, void *stream);

/* NEW.  rxq4_attention_paged_f16 over the positions of listed pages alone: each token's
 * query heads attend to the positions up to its own of the pages that `pages`
 * [n_tokens][n_kv_heads][n_select] (int32, device; rxq4_select_pages) lists for the token
 * and KV head.  Entries in any order; those that name no page with a position that the
 * token sees (-1, holes, pages behind its own) are left out; one that is there twice counts
 * twice.  n_select: 1 to 4096.  out may be q itself and overlap it in no other way, nor
 * pages.  A token that sees nothing gets zeros; what lies where a token does not look does
 * not reach its row, infinities and NaN included.  Few tokens split their lists over the
 * stream's workspace described above, by the host's sizes alone.
 * No counterpart in the reference (rxq4_attention_paged_f16). */
int rxq4_attention_selected_f16(void *out, const void *q, int n_heads, float scale,
                                const int32_t *pages, int n_select, const rxq4_seq_batch *batch,
                                const rxq4_paged_kv *cache, void *stream);

/* NEW.  The next token of each row of logits [n_rows][n_vocab] (fp32, rows
 * row_stride elements apart), from u[row] in [0, 1) (clamped to it; NaN: 0).
 * Every array but logits has one value per row in device memory; a NULL
 * parameter array leaves that parameter out.
 *   weights  w_i = exp((l_i - max l) / temperature), 64-bit; a NaN logit counts as
 *            -infinity; +infinities share the row.  temperature 0 or below (or
 *            NaN): the largest logit, lowest index, whatever else is given
 *   order    logits descending, equal ones by index ascending
 *   top_k    the first top_k of the order (0 or below: all)
 *   top_p    of those the shortest prefix whose weight is top_p of theirs (1 or
 *            above, NaN: all; the first always stays)
 *   min_p    of those the ones with w_i >= min_p (the first always stays)
 *   ids      the first of the kept whose weight and the weights before it come to
 *            more than u times the weight of all kept; -1 where every logit is
 *            -infinity or NaN
 * Results do not depend on scheduling.  Up to 48 MiB of the stream's workspace
 * (above) hold what a row's workgroups hand on.
 * No counterpart in the reference, which stops at the logits. */
int rxq4_sample_f32(int32_t *ids, const float *logits, int64_t row_stride, int n_rows,
                    int n_vocab, const float *temperature, const int32_t *top_k,
                    const float *top_p, const float *min_p, const float *u, void *stream);

/* The reference's host GEMV (gemv_quant_cpu, q4_gemm.cu:1742-1854, with its
 * callers' output rounding: fp16 at 1898, fp32 at 2016, the residual's
 * double rounding at 1941-1945), on HOST pointers only: y[M] = W[M x K] . x[K]
 * for Q4_K / Q5_K / Q6_K blocks `w`, fp16 x; y_dtype F32 or F16; a non-NULL
 * fp16 `residual` (F16 only) gives y = RNE(float(RNE(acc)) + residual).  One
 * fp32 accumulator per row in the reference's element order, bit for bit its
 * result.  The C++ API runs it for weights the GPU cannot read (no
 * weights_device alias and host-only memory) and under JLLM_FAST_GEMV=0, as
 * the reference does (q4_gemm.cu:1886-1899, 1916-1947, 1994-2016); no GPU
 * launch ever falls back to it. */
int rxq4_host_gemv(void *y, int y_dtype, const void *w, int ggml_type, const void *x,
                   const void *residual, int M, int K);

/* Number of rxq4_host_gemv computations so far in this process. */
long long rxq4_host_gemv_calls(void);

/* NEW.  Allocates the split launches' workspace for `stream` on the
 * current device now, so that no later call on that stream allocates
 * (optional; no reference counterpart, the reference splits nothing). */
int rxq4_reserve_workspace(void *stream);

/* NEW.  Synchronises `stream` and frees its workspace on the current device
 * (for hipStreamPerThread: the calling thread's); Success also when it has
 * none.  For callers that create streams per request and would otherwise
 * keep 48 MiB per stream.  A graph captured with split launches on that
 * stream must not be replayed afterwards (its partials would point at
 * freed memory); the next split launch on the stream allocates again.  No
 * reference counterpart. */
int rxq4_release_workspace(void *stream);

/* Pointer resolution of the reference (q4_gemm.cu:111-135): returns
 * w_device if non-NULL, else w if the HIP runtime reports it as device or
 * managed memory, else NULL (host-only memory cannot be read by the kernels). */
const void *rxq4_resolve_weights(const void *w, const void *w_device);

/* Library version and the reason for the last non-success status on the
 * calling thread ("" if none). */
const char *rxq4_version(void);
const char *rxq4_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
