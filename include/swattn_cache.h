/*
 * swattn_cache.h -- C ABI of libswattn.so for the 8-bit KV cache: appending
 * and reading rows, routed decode over it, sums of attention weights, and
 * eviction by them.  The conventions are those of swattn.h: device pointers, a
 * hipStream_t passed as void*, no allocation, no synchronisation, the same
 * status codes and swattn_last_error().  Nothing here has a counterpart in
 * the reference, which is prefill-only and keeps no cache.
 *
 * The cache of one layer:
 *   k, v                codes [batch, cache_len, heads_kv, 128], one byte each
 *                       (SWATTN_CODE_*), 16-byte aligned
 *   k_scales, v_scales  fp32 [batch, heads_kv, ceil(cache_len / block)]: cached
 *                       row r of KV head h stands for code * scale[b][h][r / block]
 *   block               tokens that share a scale: 16, 32, 64 or 128
 * Row r of a sequence is valid where r < cache_lens[b] (int32 on the device,
 * clamped to [0, cache_len] by every entry point).  What lies behind is never
 * looked at, scales of blocks without a valid row included.
 *
 * Scales that these entry points write are powers of two: for a block's
 * largest magnitude a, the smallest 2^e >= 2^-100 with a <= qmax * 2^e (qmax
 * 448 for e4m3, 127 for int8), so that scaling is exact and a value is rounded
 * once, to the nearest code, ties to even.  Where that code would stand for
 * more than the largest bf16 number (from 248 * 2^120 on for e4m3, 63.5 *
 * 2^122 for int8) the next smaller one is taken: finite values read as finite
 * ones.  A block that takes a NaN or an
 * infinity gets scale NaN: its rows read as NaN until all of them are gone.
 * Caches with other (positive, finite) scales, made elsewhere, may be read,
 * attended, appended to and evicted from.
 */
#ifndef SWATTN_CACHE_H_
#define SWATTN_CACHE_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SWATTN_CODE_E4M3 0   /* OCP fp8: sign, 4 exponent and 3 mantissa bits, no infinities */
#define SWATTN_CODE_INT8 1   /* two's complement; -128 is read, and written only where a begun
                              * block that holds it takes a slightly larger scale */

/*
 * Append new rows to the sequences of a cache.
 *
 *   new_k, new_v  bf16 rows [.., heads_kv, 128].  cu_seqlens NULL: [batch,
 *                 rows, ..], of which sequence b appends the first
 *                 counts[b] (clamped to [0, rows]; counts NULL: all).  With
 *                 cu_seqlens (batch + 1 ascending int32 offsets on the device,
 *                 clamped to [0, total_rows]): packed [total_rows, ..];
 *                 sequence b appends rows cu_seqlens[b] .. cu_seqlens[b + 1]
 *                 - 1, at most `rows` of them.
 *   cache_lens    valid rows before the call; the new rows follow them.  Rows
 *                 that would lie behind cache_len are dropped.
 *   lens_out      int32 [batch]: valid rows after the call (min with cache_len).
 *                 May not alias cache_lens.
 * A block that held valid rows keeps its scale if the new rows fit it, or
 * takes theirs, and its rows are rounded again to that.  Rows behind the new
 * end keep their codes.  Sequences must not overlap in memory.
 */
int swattn_cache_append(const void* new_k, const void* new_v, const int32_t* cu_seqlens,
                        const int32_t* counts, const int32_t* cache_lens, void* k, void* v,
                        float* k_scales, float* v_scales, int32_t* lens_out, int32_t batch,
                        int64_t rows, int64_t total_rows, int64_t cache_len, int32_t heads_kv,
                        int32_t head_dim, int32_t block, int32_t code, void* stream);

/*
 * Read `rows` rows per sequence as bf16 [batch, rows, heads_kv, 128], from
 * row starts[b] (starts NULL: from row `start` in every sequence).  Rows
 * outside [0, cache_lens[b]) (cache_lens NULL: [0, cache_len)) come out as 0.
 * rows * heads_kv below 2^28.
 */
int swattn_cache_read(const void* k, const void* v, const float* k_scales, const float* v_scales,
                      const int32_t* starts, int64_t start, const int32_t* cache_lens, void* out_k,
                      void* out_v, int32_t batch, int64_t rows, int64_t cache_len,
                      int32_t heads_kv, int32_t head_dim, int32_t block, int32_t code,
                      void* stream);

/*
 * swattn_decode_fwd over an 8-bit cache: same rule, arguments and results
 * (bf16 O, fp32 log2 LSE; a sequence with no key gets O = NaN, LSE = -inf).
 *   key_weights  fp32 [batch, heads_kv, cache_len], or NULL.  Added to: for
 *                each key that the new token attends, the sum over the KV
 *                head's query heads of its softmax weight 2^(s - LSE).  Other
 *                entries keep their value.
 *   workspace    >= swattn_cache_decode_workspace_bytes(..., key_weights !=
 *                NULL), asked on the current device; 256-byte aligned.  With
 *                key_weights it also holds the call's scores, fp32 [batch,
 *                heads_q, cache_len rounded up to 32].
 */
size_t swattn_cache_decode_workspace_bytes(int32_t batch, int64_t cache_len, int32_t heads_q,
                                           int32_t heads_kv, int32_t with_weights);
int swattn_cache_decode_fwd(const void* q, const void* k, const void* v, const float* k_scales,
                            const float* v_scales, const int32_t* cache_lens, const uint8_t* full,
                            void* out, float* lse, float* key_weights, int32_t batch,
                            int64_t cache_len, int32_t heads_q, int32_t heads_kv,
                            int32_t head_dim, int32_t window, int32_t block, int32_t code,
                            float scale_log2, void* workspace, size_t workspace_bytes,
                            void* stream);

/*
 * The attention weight that each key received from a prefill's queries:
 *   key_weights[b][h][j] = sum over listed rows r that may see key j and over
 *                          the query heads of KV head h of 2^(c q_r.k_j - LSE_r)
 * (0 for a key that no row sees).  q, k, the lists, the metadata bounds, the
 * shapes, window and scale_log2 are those of swattn_prefill_fwd and lse is its
 * result.  Each list's key bounds must be non-decreasing along the list, as
 * for swattn_prefill_bwd.  A row with LSE +inf and finite scores adds nothing.
 * scale_log2 must be finite, and batch * seq_q * heads_q below 2^31.
 *   key_weights  fp32 [batch, heads_kv, seq_kv]; every entry is written
 *   workspace    >= swattn_prefill_key_weights_workspace_bytes(), 256-byte aligned
 */
size_t swattn_prefill_key_weights_workspace_bytes(int32_t batch, int64_t seq_kv, int32_t heads_q,
                                                  int32_t heads_kv, int32_t head_dim,
                                                  int64_t n_full, int64_t n_local);
int swattn_prefill_key_weights(const void* q, const void* k, const float* lse,
                               const int32_t* full_idx, int64_t n_full, const int32_t* local_idx,
                               int64_t n_local, const int32_t* full_starts,
                               const int32_t* local_starts, const int32_t* causal_ends,
                               float* key_weights, int32_t batch, int64_t seq_q, int64_t seq_kv,
                               int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                               int32_t window, float scale_log2, void* workspace,
                               size_t workspace_bytes, void* stream);

/*
 * Evict: copy what a budget keeps of each sequence into another cache.  For a
 * sequence of n = cache_lens[b] rows and each KV head on its own: all rows if
 * n <= budget, else the newest `recent` rows and those budget - recent of the
 * older ones with the largest key_weights (NaN counts as largest; of equal
 * weights the lower row first).  Kept rows stay in their order, at rows 0 ..
 * of the destination; each destination block gets the scale of its rows and
 * they are rounded to that.
 *   out_*        the destination, out_len >= budget rows per sequence, of the
 *                same heads, block and code; may overlap no input
 *   out_weights  fp32 [batch, heads_kv, out_len]: the kept rows' weights, 0 in
 *                all rows behind
 *   lens_out     int32 [batch]: min(n, budget)
 *   workspace    >= swattn_cache_evict_workspace_bytes(), 256-byte aligned
 */
size_t swattn_cache_evict_workspace_bytes(int32_t batch, int32_t heads_kv, int64_t budget);
int swattn_cache_evict(const void* k, const void* v, const float* k_scales, const float* v_scales,
                       const float* key_weights, const int32_t* cache_lens, void* out_k,
                       void* out_v, float* out_k_scales, float* out_v_scales, float* out_weights,
                       int32_t* lens_out, int32_t batch, int64_t cache_len, int64_t out_len,
                       int32_t heads_kv, int32_t head_dim, int32_t block, int32_t code,
                       int64_t budget, int64_t recent, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}  // extern "C"
#endif

#endif  // SWATTN_CACHE_H_
