/*
 * MI355X (gfx950) split-K decode attention over vLLM's int8 per-token-head paged KV cache.
 *
 * C ABI of libpthdec.so. Plain pointers, strides and sizes only; every device pointer is
 * owned by the caller and no entry point allocates, frees or synchronises the host, so a
 * launch may be captured in a HIP graph.
 *
 * Cache row layout (one row per (block, slot, kv head), 520 bytes):
 *     [ K int8 x 256 | k_scale f32 | V int8 x 256 | v_scale f32 ]
 * key_cache is the int8 view [blocks, block_size, Hkv, 260] whose last dim is contiguous;
 * value_cache is the same storage shifted by 260 bytes; k_scale / v_scale are f32 views
 * [blocks, block_size, Hkv] at +256 / +516 bytes of each row.
 *
 * Range of the attention entry points (decode and prefill): each key's value weight is formed in
 * fp16 as p * v_scale * 16 with p <= 16 (the running max lags a row's true max by at most 4 in
 * log2 units), so v_scale must stay below 255.9, i.e. V rows with absmax below ~32,500. Larger
 * scales can overflow that weight to infinity. pth_cache_write produces such scales only from
 * V inputs above ~32,500 in magnitude.
 *
 * Reference interfaces replaced (paths relative to the 0c33/mi50-vllm-lab tree):
 *   pth_dec_launch             <- kernels/pth_dec/pth_dec.cu:285-314 (same signature)
 *   pth_dec_launch_window      <- same, plus the window / non-causal rule of
 *                                 patches/vllm/gfx906_fa_paged.patch:7-20 and
 *                                 kernels/fa_pth/kernel/fattn-q8-paged.cuh:219-229
 *   pth_dec_supported_layout   <- supported_layout, kernels/pth_dec/pth_dec.cpp:25-41
 *   pth_dec_decode             <- decode, kernels/pth_dec/pth_dec.cpp:43-91 (the torch op body,
 *                                 with tensors passed as pd_tensor descriptors)
 *   pth_fa_forward             <- forward_pth, kernels/fa_pth/pth_fa.cpp:41-85 (chunked prefill)
 *   pth_cache_write            <- vLLM's int8 per-token-head cache update (do_kv_cache_update)
 */
#ifndef PTH_DEC_H
#define PTH_DEC_H

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* dtype codes used in pd_tensor.dtype */
#define PD_DTYPE_INT8 1
#define PD_DTYPE_FP16 2
#define PD_DTYPE_FP32 3
#define PD_DTYPE_INT32 4
#define PD_DTYPE_BF16 5
#define PD_DTYPE_INT64 6

#define PD_MAX_DIMS 4

/* A strided tensor view: data pointer, dtype code, rank, sizes and strides in elements. */
typedef struct pd_tensor {
    const void* data;
    int32_t dtype;
    int32_t ndim;
    int64_t sizes[PD_MAX_DIMS];
    int64_t strides[PD_MAX_DIMS];
} pd_tensor;

/*
 * Split-K decode attention, causal, no window. Same arguments, meaning and error codes as
 * kernels/pth_dec/pth_dec.cu:285-290:
 *   q            fp16 [num_tokens, heads_q, 256], token stride q_st elements, head stride 256
 *   kc           int8 cache base (key_cache.data_ptr()); k_sb / k_ss / k_sh are the byte strides
 *                of blocks, slots and kv heads; V sits at +260 bytes of each K row
 *   block_table  int32, row stride bt_stride; seq_lens int32 [num_seqs];
 *   qsl          int32 query_start_loc [num_seqs + 1]
 *   part_o       fp32 [>= num_tokens, heads_q, nseg, 256]; part_m / part_l fp32 [.., heads_q, nseg]
 *   out          fp16, element (t, h, d) at out + t * o_st + h * o_sh + d
 * Returns hipErrorInvalidValue unless heads_q == 6 * heads_kv, 1 <= qmax <= 4,
 * 1 <= nsplit <= nseg and num_seqs >= 1.
 * Here and in the other entries that run both kernels, a batch of several sequences for which
 * nsplit * heads_kv * num_seqs is above the CU count (and nsplit >= 2, at most 32 rows per kv head, and
 * min(nseg, 128) > nsplit + nsplit / 8 or nsplit >= 16) is dealt evenly over the GPU by seq_lens instead: it
 * may then use up to min(nseg, 128) segments of the partial buffers rather than nsplit of them.
 */
hipError_t pth_dec_launch(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                          const int* block_table, int bt_stride, const int* seq_lens, const int* qsl,
                          int num_seqs, int num_tokens, int heads_q, int heads_kv, int block_size,
                          float scale, int qmax, float* part_o, float* part_m, float* part_l, int nseg,
                          int nsplit, void* out, long o_st, long o_sh, hipStream_t stream);

/*
 * pth_dec_launch with the arguments the DFlash2 drafter needs appended:
 *   window  > 0: row j of a sequence (absolute position p_j = seq_len - q_len + j) sees key k
 *                only if p_j - k < window; <= 0 (e.g. -1): no window
 *   causal  != 0: key k > p_j is masked; 0: every key < seq_len is visible (non-causal block)
 * Any GQA ratio heads_q / heads_kv with qmax * (heads_q / heads_kv) <= 48 is accepted
 * (MTP 4 x 6 = 24 rows, DFlash2 8 x 6 = 48 rows).
 */
hipError_t pth_dec_launch_window(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                 const int* block_table, int bt_stride, const int* seq_lens,
                                 const int* qsl, int num_seqs, int num_tokens, int heads_q, int heads_kv,
                                 int block_size, float scale, int qmax, float* part_o, float* part_m,
                                 float* part_l, int nseg, int nsplit, void* out, long o_st, long o_sh,
                                 hipStream_t stream, int window, int causal);

/*
 * The two stages of pth_dec_launch_window launched separately (no counterpart in the
 * reference, which always launches both): the split-K partial pass writes part_o / part_m /
 * part_l, the combine pass merges them into out. Same argument checks.
 */
hipError_t pth_dec_launch_partial(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                  const int* block_table, int bt_stride, const int* seq_lens,
                                  const int* qsl, int num_seqs, int num_tokens, int heads_q,
                                  int heads_kv, int block_size, float scale, int qmax, float* part_o,
                                  float* part_m, float* part_l, int nseg, int nsplit,
                                  hipStream_t stream, int window, int causal);
hipError_t pth_dec_launch_combine(const int* seq_lens, const int* qsl, int num_seqs, int num_tokens,
                                  int heads_q, int qmax, const float* part_o, const float* part_m,
                                  const float* part_l, int nseg, int nsplit, void* out, long o_st,
                                  long o_sh, hipStream_t stream);

/*
 * pth_dec_launch_window without the partial buffers, for callers that cannot allocate (code
 * under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). No
 * counterpart in the reference. The split partials go to a device array the library holds (32 MiB
 * per GPU, for the life of the process); this call allocates nothing. Limit:
 * num_tokens * heads_q * nsplit * 1032 bytes <= 32 MiB (e.g. 4 tokens x 24 heads x 64 splits);
 * beyond it the call returns hipErrorOutOfMemory and launches nothing. Other checks and errors
 * as pth_dec_launch_window. Every call on a GPU shares that GPU's array: calls that overlap on
 * one GPU (different streams) race; calls on one stream are ordered and safe.
 */
hipError_t pth_dec_launch_noalloc(const void* q, int q_st, const void* kc, int k_sb, int k_ss, int k_sh,
                                  const int* block_table, int bt_stride, const int* seq_lens,
                                  const int* qsl, int num_seqs, int num_tokens, int heads_q,
                                  int heads_kv, int block_size, float scale, int qmax, int nsplit,
                                  void* out, long o_st, long o_sh, hipStream_t stream, int window,
                                  int causal);

/* 1 if the four cache views have the row layout above, else 0 (pth_dec.cpp:25-41). */
int pth_dec_supported_layout(const pd_tensor* key_cache, const pd_tensor* value_cache,
                             const pd_tensor* k_scale, const pd_tensor* v_scale);

/*
 * The torch op `decode` of kernels/pth_dec/pth_dec.cpp:49-91 over descriptors, with window
 * and causal appended. Validates every tensor like the reference's TORCH_CHECKs (and refuses
 * sizes, counts or a window that do not fit in 32 bits); on failure
 * returns 1 and writes the reference's message into err (errlen bytes, NUL-terminated);
 * returns 2 with the HIP error string if the launch fails; 0 on success.
 */
int pth_dec_decode(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                   const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                   const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out,
                   double scale, const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l,
                   int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window, int64_t causal,
                   hipStream_t stream, char* err, int errlen);

/*
 * pth_dec_decode that also stores each row's softmax logarithm, for callers that need the weights of single keys
 * (pth_cache_key_weights) or merge the result with attention over other keys. No counterpart in the reference.
 *   lse          fp32, contiguous [>= T, Hq]: ln(sum over the visible keys of e^(scale q . k)), -inf for a row
 *                that sees no key; rows that out does not get are left alone
 */
int pth_dec_decode_lse(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                       const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                       const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out,
                       double scale, const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l,
                       const pd_tensor* lse, int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window,
                       int64_t causal, hipStream_t stream, char* err, int errlen);

/*
 * pth_dec_decode for rows that see a sliding window and a few first keys, which stay visible however long the sequence grows. No
 * counterpart in the reference.
 *   lse          null, or as for pth_dec_decode_lse
 *   sinks        >= 0: row j (absolute position p_j) sees key k < seq_len, k <= p_j where causal, if p_j - k < window or k < sinks;
 *                without a window (<= 0) every row sees those keys anyway
 * Pages in which no row of the sequence sees a key are not addressed: their table entries may name anything. A key whose scale is not
 * finite makes the rows that see it so and no others. Other arguments, checks and return codes are those of pth_dec_decode.
 */
int pth_dec_decode_sinks(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                         const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out,
                         double scale, const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l,
                         const pd_tensor* lse, int64_t num_seqs, int64_t qmax, int64_t nsplit, int64_t window,
                         int64_t sinks, int64_t causal, hipStream_t stream, char* err, int errlen);

/*
 * Decode attention of a batch whose sequences share their first prefix_len keys (a common prompt or document, samples of
 * one prompt): pth_dec_decode's causal attention without window, with the shared keys read once for the whole batch. No
 * counterpart in the reference.
 *   q .. part_l, num_seqs, qmax   as for pth_dec_decode; at least 4 segments in the partial buffers
 *   lse          null, or as for pth_dec_decode_lse
 *   prefix_len   >= 0, within the block table; the tables of the sequences that hold the prefix and their query tokens
 *                behind it (seq_len - q_len >= prefix_len) name the same keys for it (the same blocks, or for a block that
 *                the prefix ends in, blocks that agree on its keys): the table of the first such sequence is
 *                read. Sequences that do not are computed from their own table alone.
 * At most 2^25 (token, head) rows and 2^30 / heads_kv key tiles that the block table can hold. The weights
 * enter P.V as the decode's hi + lo. Returns 0, 1 or 2 as above.
 */
int pth_dec_decode_shared(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                          const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                          const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* out,
                          double scale, const pd_tensor* part_o, const pd_tensor* part_m, const pd_tensor* part_l,
                          const pd_tensor* lse, int64_t num_seqs, int64_t qmax, int64_t prefix_len,
                          hipStream_t stream, char* err, int errlen);

/* Library version string. */
const char* pth_dec_version(void);

/*
 * Causal chunked prefill over the same int8 per-token-head cache. Replaces forward_pth,
 * kernels/fa_pth/pth_fa.cpp:41-85 (same arguments, meaning and error messages), with the output
 * passed in instead of allocated:
 *   q            fp32 [B, Hq, Sq, 256] contiguous; query token i of sequence b sits at absolute
 *                position q_abs_offset[b] + i and sees keys k <= that position, k < seq_lens[b]
 *   key_cache / value_cache  the cache views (value_cache = key_cache + 260 bytes)
 *   block_table  int32 [B, max_blocks]; seq_lens, q_abs_offset int32 [B]
 *   out          fp32 [B, Sq, Hq, 256], unit dim stride
 * Q is rounded to fp16 for the matrix cores; scores and P.V accumulate in fp32. B, Hq and Sq
 * must be below 2^31. Returns 0, 1 (validation failure, message in err) or 2 (launch failure).
 * Accuracy: each softmax weight enters P.V as one fp16 P' = p * v_scale * 16 (11 significant
 * bits), so an output element is within 2e-3 + 2^-11 * sum_k p_k |v_k| / l of the float64
 * result (v_k the dequantised value, l = sum_k p_k). On caches of N(0,1)-like rows that is
 * inside max-abs 2e-3 / mean-abs 2e-4; on caches with outlier rows (1 % of rows at 50x) the
 * second term dominates (max-abs 5.1e-2 at outputs near 148, 2^-11.5 relative). That is below
 * one fp16 spacing of the output, so a caller that stores fp16 (vLLM's attention output) loses
 * nothing to it; a caller that needs fp32-grade results on such caches uses
 * pth_fa_forward_exact.
 */
int pth_fa_forward(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                   const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                   const pd_tensor* q_abs_offset, const pd_tensor* out, hipStream_t stream, char* err,
                   int errlen);

/*
 * No counterpart in the reference. pth_fa_forward with the decode's numerics: K and V converted
 * to fp16 without the widening bias, so the fp32 accumulators hold only the products' own sums,
 * and P' carried as fp16 hi + lo (~22 bits instead of 11). It is for callers whose caches hold rows
 * with very large scales (attention sinks, outlier tokens), where pth_fa_forward's single-fp16
 * P' can miss max-abs 2e-3. It is slower: the P.V products double. Arguments, checks, errors and
 * return codes are those of pth_fa_forward.
 */
int pth_fa_forward_exact(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                         const pd_tensor* q_abs_offset, const pd_tensor* out, hipStream_t stream, char* err,
                         int errlen);

/*
 * No counterpart in the reference. pth_fa_forward (exact != 0: pth_fa_forward_exact) with each
 * query tile's keys split over nsplit workgroups, for chunks too short to fill the GPU (a
 * workgroup takes 192 query rows of one kv head, so a 64-token chunk of 24 q / 4 kv heads
 * launches 8 of them per split) or whose workgroups end in a part-filled round. Each split stores unnormalised partials in the caller's
 * workspace, and a second kernel merges them into out.
 *   workspace  fp32, contiguous, 16-byte aligned, at least B * Sq * Hq * nsplit * 258 floats
 *              (ignored when nsplit == 1)
 *   nsplit     1..64; when above 1, B * Sq * Hq must be below 2^31
 * Other arguments, checks, errors and return codes are those of pth_fa_forward. The results
 * equal pth_fa_forward's within rounding (the partial sums are merged in another order).
 */
int pth_fa_forward_split(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                         const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                         const pd_tensor* q_abs_offset, const pd_tensor* out, const pd_tensor* workspace,
                         int64_t nsplit, int64_t exact, hipStream_t stream, char* err, int errlen);

/*
 * No counterpart in the reference. The prefill with the key tiles of all query tiles dealt evenly over the GPU by
 * the lengths on the device, for chunks whose query tiles see different numbers of keys (fresh prompts), do not
 * fill the GPU, or belong to several sequences. Two forms:
 *   query_start == NULL: pth_fa_forward's arguments, checks and messages (num_seqs is ignored).
 *   query_start (host, int[num_seqs + 1], num_seqs <= 32): q fp16 [T, Hq, 256] with unit dim stride, rows
 *     16-byte aligned; sequence i has rows [query_start[i], query_start[i + 1]) of q and out, the last tokens
 *     of its seq_lens[i] keys; block_table and seq_lens have a row per sequence; out fp16 [T, Hq, 256],
 *     rows 8-byte aligned, T its own (both hold the sequences' rows). The rows outside the sequences are left alone. q_abs_offset is ignored.
 *   workspace  fp32, contiguous, 16-byte aligned, of pth_fa_balanced_workspace floats (fewer, down to
 *              2 x 192 x 258, only lower the number of workgroups)
 *   max_keys   a bound on the keys any row sees, to size the launch; a wrong one costs time only
 *   nsplit     0; or, in the rows form with one sequence, 1..64: pth_fa_forward_split's kernels on the rows
 *              instead (workspace rows x Hq x nsplit x 258 floats when above 1)
 * Numerics and return codes are those of pth_fa_forward (exact != 0: pth_fa_forward_exact); the results equal
 * theirs within rounding (partial sums are merged in another order).
 */
int pth_fa_forward_balanced(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                            const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                            const pd_tensor* q_abs_offset, const int* query_start, int64_t num_seqs, const pd_tensor* out,
                            const pd_tensor* workspace, int64_t max_keys, int64_t nsplit, int64_t exact, hipStream_t stream,
                            char* err, int errlen);
/* Workspace floats for pth_fa_forward_balanced on the current device; 0 if it does not take such a call (no query
 * tokens, more than 32 sequences in the rows form, more than 2^31 key tiles). table_keys: block_table columns x
 * block size. */
int64_t pth_fa_balanced_workspace(int64_t num_seqs, const int* query_start, int64_t sq, int64_t heads_q, int64_t heads_kv,
                                  int64_t max_keys, int64_t table_keys);

/*
 * Causal chunked prefill of rows that see a sliding window and a few first keys. No counterpart in the reference.
 *   q, out       fp16 [T, Hq, 256], unit dim stride, rows of q 16-byte and of out 8-byte aligned; out and the workspace
 *                must not overlap each other, q, the cache or the tables
 *   query_start_loc  int32 [>= num_seqs + 1], device: sequence i has rows [query_start_loc[i], query_start_loc[i + 1]) of q and out, the last
 *                tokens of its seq_lens[i] keys (block_table and seq_lens have a row per sequence). Rows outside the sequences, and of
 *                sequences of no keys, are left alone
 *   window >= 1, sinks >= 0   the row at position p sees key k <= p if p - k < window or k < sinks
 *   nsplit       1..64: key splits per query tile (256 or 128 rows of one kv head, as the sizes suggest); pth_fa_window_splits' count
 *                suits the sizes
 *   workspace    fp32, contiguous, 16-byte aligned, of T * Hq * nsplit * 258 floats (null or ignored when nsplit is 1)
 *   exact        0: each softmax weight enters P.V as one fp16; else as fp16 hi + lo. K and V are widened exactly in both
 * Pages in which no row of a query tile sees a key are not addressed for it: the table's entries for pages between the sinks and
 * the first row's window may name anything. A key whose scale is not finite makes the rows that see it so and no others. Returns 0, 1
 * or 2 as above.
 */
int pth_fa_forward_window(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                          const pd_tensor* block_table, const pd_tensor* seq_lens, double scale,
                          const pd_tensor* query_start_loc, const pd_tensor* out, const pd_tensor* workspace, int64_t num_seqs,
                          int64_t window, int64_t sinks, int64_t nsplit, int64_t exact, hipStream_t stream, char* err,
                          int errlen);
/* Splits that such a call is rated fastest with on the current device; table_keys: block_table columns x block size. */
int64_t pth_fa_window_splits(int64_t tokens, int64_t num_seqs, int64_t heads_q, int64_t heads_kv, int64_t window,
                             int64_t sinks, int64_t table_keys, int64_t exact);

/*
 * KV-cache writer and quantiser: the producer of the 520-byte rows the two operators read.
 * Replaces vLLM's cache update for int8 per-token-head KV, which the reference calls as
 * do_kv_cache_update(layer, key, value, kv_cache, slot_mapping)
 * (upstream/pr-dflash2/0002-fix-gfx906-keep-the-drafter-s-sliding-window-in-the-.patch:81-87;
 * the update itself lives in the un-vendored vLLM fork KIntegrated/vllm-gfx906-mobydick 0.30.0).
 *   key, value   fp16, bf16 or fp32 [T, Hkv, 256], unit dim stride
 *   key_cache, value_cache, k_scale, v_scale   the cache views (as for pth_dec_decode)
 *   slot_mapping int64 [T]: slot = block * block_size + offset; negative slots (padding) and
 *                slots past the cache are skipped
 * Per (token, kv head): scale = absmax / 127 (0 for an all-zero row), q = clamp(rint(x / scale),
 * -127, 127) with x / scale correctly rounded. At most 2^30 (token, kv head) rows per call.
 * Returns 0, 1 (validation failure, message in err) or 2 (launch failure).
 */
int pth_cache_write(const pd_tensor* key, const pd_tensor* value, const pd_tensor* key_cache,
                    const pd_tensor* value_cache, const pd_tensor* k_scale, const pd_tensor* v_scale,
                    const pd_tensor* slot_mapping, hipStream_t stream, char* err, int errlen);

/*
 * Rotary positions and the cache write of a layer's new tokens in one launch. No counterpart in the reference, whose
 * engine runs its own rotary kernel before the cache update.
 *   query        fp16, bf16 or fp32 [T, Hq, 256], unit dim stride; rotated into query_out
 *   query_out    [T, Hq, 256] of the query's dtype or fp16: the query itself (same data, dtype and strides: in place) or
 *                a tensor that does not overlap it; its rows apart, and no part of key or value. (Views of one buffer are
 *                known to be apart by their extents, or by a stride that both have.)
 *   key, value   [T, Hkv, 256] of the query's dtype, left as they are; the rotated key and the value are
 *                quantised into the cache rows as pth_cache_write does
 *   positions    int64 [>= T]; a token whose position lies outside cos_sin is skipped (query_out and cache row stay)
 *   cos_sin      fp32 [positions, rotary_dim], rotary_dim a multiple of 8 up to 256: cosines of the
 *                rotary_dim / 2 angles, then sines
 *   interleaved  0: pair i is dims (i, i + rotary_dim / 2); else (2 i, 2 i + 1); the dims from rotary_dim on stay
 *   slot_mapping int64 [>= T]; tokens with a slot below 0 or past the cache write no row (their query is rotated). No two
 *                tokens of a call may have the same slot
 * Rotation and quantisation are fp32, each product and sum rounded; the rotated key is not rounded to its dtype
 * first. Rows are aligned to four elements. Returns 0, 1 (validation failure, message in err) or 2 (launch failure).
 */
int pth_cache_write_rotary(const pd_tensor* query, const pd_tensor* query_out, const pd_tensor* key,
                           const pd_tensor* value, const pd_tensor* positions, const pd_tensor* cos_sin,
                           const pd_tensor* key_cache, const pd_tensor* value_cache, const pd_tensor* k_scale,
                           const pd_tensor* v_scale, const pd_tensor* slot_mapping, int64_t interleaved,
                           hipStream_t stream, char* err, int errlen);

/*
 * Running attention weights of the cached keys: adds to weights[b, g, t] the softmax weight that the query rows of
 * sequence b and kv head g gave key t, sum over rows of e^(scale q . k_t - lse). No counterpart in the reference.
 *   q, key_cache .. query_start_loc, scale, num_seqs, qmax   as for pth_dec_decode (causal, no window)
 *   lse          fp32, contiguous [>= T, Hq], of pth_dec_decode_lse or _shared on the same rows; a row of
 *                -inf adds nothing
 *   weights      fp32 [>= num_seqs, Hkv, keys <= 2^28], unit key stride, its rows apart; only keys below seq_len and below `keys`
 *                are touched
 * Every weight is formed in a fixed order (no atomics). Returns 0, 1 or 2 as above.
 */
int pth_cache_key_weights(const pd_tensor* q, const pd_tensor* key_cache, const pd_tensor* value_cache,
                    const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
                    const pd_tensor* seq_lens, const pd_tensor* query_start_loc, const pd_tensor* lse,
                    const pd_tensor* weights, double scale, int64_t num_seqs, int64_t qmax, hipStream_t stream,
                    char* err, int errlen);

/*
 * Eviction by running weights: per sequence and kv head the last `recent` keys and the keep - recent others with the
 * largest weights stay (equal weights: the lowest key; NaN counts as the largest), in the order of their positions. Their
 * rows are copied into the blocks of new_block_table; the old blocks are left as they are. No counterpart in the reference.
 *   weights      fp32 [>= num_seqs, Hkv, keys <= 2^28]. A sequence is taken to end where its weights or its block table do: n =
 *                min(seq_len, keys, keys of the table), and its keys behind n, the newest ones, are dropped. `keys` must hold
 *                the longest sequence for `recent` to be its last keys
 *   block_table, seq_lens   int32, the batch before; sequences of at most keep keys are copied whole
 *   new_block_table         int32 [>= num_seqs, columns for keep keys]: blocks that no table row of the call reads
 *                           and no two of its rows share, in the part that holds a sequence's min(n, keep) keys
 *   new_seq_lens            int32 [>= num_seqs], written: min(n, keep)
 *   new_weights             fp32 [>= num_seqs, Hkv, >= keep], written: the kept keys' weights, then zeros
 *   kept                    int32, contiguous [>= num_seqs, Hkv, keep], written: the kept keys' numbers, then -1
 *   keep, recent            1 <= keep <= 2^28, 0 <= recent <= keep
 * The new tensors must not be the old ones, and those written (new_seq_lens, new_weights, kept) overlap neither what is
 * read nor each other. Rotated keys keep the positions they were rotated by; rows written later take
 * positions (pth_cache_write_rotary) that count the evicted keys too. Returns 0, 1 or 2 as above.
 */
int pth_cache_evict(const pd_tensor* weights, const pd_tensor* key_cache, const pd_tensor* value_cache,
              const pd_tensor* k_scale, const pd_tensor* v_scale, const pd_tensor* block_table,
              const pd_tensor* seq_lens, const pd_tensor* new_block_table, const pd_tensor* new_seq_lens,
              const pd_tensor* new_weights, const pd_tensor* kept, int64_t num_seqs, int64_t keep, int64_t recent,
              hipStream_t stream, char* err, int errlen);

/*
 * pth_cache_write_rotary with the norms that a model applies to its query and key heads before the rotation: every head x of
 * query and key is x / sqrt(mean(x^2) + eps) * (weight + weight_offset) first, in fp32. No counterpart in the reference.
 *   query_weight, key_weight   contiguous [256], both fp32 or both of the query's dtype, aligned to 4 elements
 *   eps, weight_offset         eps >= 0
 * The other arguments are pth_cache_write_rotary's; query_out must not overlap the weights either. In place the whole query
 * is written. Returns 0, 1 or 2 as above.
 */
int pth_cache_write_norm_rotary(const pd_tensor* query, const pd_tensor* query_out, const pd_tensor* key,
                                const pd_tensor* value, const pd_tensor* query_weight, const pd_tensor* key_weight,
                                double eps, double weight_offset, const pd_tensor* positions, const pd_tensor* cos_sin,
                                const pd_tensor* key_cache, const pd_tensor* value_cache, const pd_tensor* k_scale,
                                const pd_tensor* v_scale, const pd_tensor* slot_mapping, int64_t interleaved,
                                hipStream_t stream, char* err, int errlen);

/*
 * Block tables and reference counts on the device. No counterpart in the reference, whose engine keeps them on the host.
 *   caches       `layers` (1..128) raw caches, int8 [pages <= 2^22, Hkv, block_size, 520], of the same sizes and strides, their rows
 *                8-byte aligned and apart, also from other caches' and the other tensors (one given twice counts once); page
 *                numbers are those of all of them
 *   refs         int32 [pages], how many table entries name each page; 0 (or less): the page is free
 *   block_table  int32 [B, columns], an entry outside [0, pages) names no page
 *   workspace    int32, 16-byte aligned, of pth_cache_pages_workspace(pages, B, N) (0, 0 for compact); its contents need not be
 *                kept between calls, and calls that may overlap in time need one each
 *
 * pth_cache_fork_pages: row i of the new tables goes on from row p = parents[i] (null: i) of n = seq_lens[p] keys. Of
 * its columns below ceil((n + grow) / block_size), those of full pages keep p's entry, or become -1 if window > 0 and all keys of the
 * page lie at or past `sinks` and before n + 1 - window; each other column keeps p's entry if the row is the first child
 * of p and the page's count is 1, else it takes a free page (the lowest of those free before the call, in the order of row and
 * column), and the keys below n that p has there are copied for all caches. All further columns become -1. The old rows'
 * references are dropped, the new rows' counted.
 *   seq_lens     int32 [B] (less than 0 counts as 0); parents int32 [N] or null; a parent outside [0, B): an empty row of length 0
 *   new_refs     int32 [pages]: refs itself, or apart from it
 *   new_block_table, new_seq_lens   int32 [N, columns] and [N]: apart from the old ones, without parents also the old ones
 *                themselves
 *   needed       int32 [1], written: the pages wanted. Where more than were free, the last columns that wanted one are -1
 *   grow, sinks  >= 0; window <= 0: none
 * At most 8,192 rows in either table and 2^31 - 1 entries in the new one; new_refs of a page that is free is 0.
 *
 * pth_cache_compact_pages: of n used pages, those numbered n or above move, in order, into the free ones below n, for all caches.
 *   new_refs, new_block_table   as above, each the old one or apart from it; an entry that names no used page becomes -1
 *   places       int32 [pages], written: where each page lies now, -1 for a free one
 *   used         int32 [1], written: n
 *
 * The tensors that are written overlap neither each other nor those that are read, but for what is said above. No results depend
 * on the order in which the device works. Both return 0, 1 or 2 as above.
 */
int pth_cache_fork_pages(const pd_tensor* caches, int64_t layers, const pd_tensor* refs, const pd_tensor* block_table,
                         const pd_tensor* seq_lens, const pd_tensor* parents, const pd_tensor* new_refs,
                         const pd_tensor* new_block_table, const pd_tensor* new_seq_lens, const pd_tensor* needed,
                         const pd_tensor* workspace, int64_t grow, int64_t window, int64_t sinks, hipStream_t stream,
                         char* err, int errlen);
int pth_cache_compact_pages(const pd_tensor* caches, int64_t layers, const pd_tensor* refs, const pd_tensor* block_table,
                            const pd_tensor* new_refs, const pd_tensor* new_block_table, const pd_tensor* places,
                            const pd_tensor* used, const pd_tensor* workspace, hipStream_t stream, char* err, int errlen);
/* Workspace int32s of the above for caches of `pages` pages and tables of `rows` old and `new_rows` new rows; 0 if out of range. */
int64_t pth_cache_pages_workspace(int64_t pages, int64_t rows, int64_t new_rows);

#ifdef __cplusplus
}
#endif

#endif /* PTH_DEC_H */
