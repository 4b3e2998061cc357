/*
 * swattn_shared.h -- C ABI of libswattn.so for a decode step of sequences that continue
 * shared prefixes.  The conventions are those of swattn.h: device pointers, a
 * hipStream_t passed as void*, no allocation, no synchronisation, the same status codes
 * and swattn_last_error().  Nothing here has a counterpart in the reference, which is
 * prefill-only.
 */
#ifndef SWATTN_SHARED_H_
#define SWATTN_SHARED_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SWATTN_SHARED_MAX_SEQS 1024
#define SWATTN_SHARED_MAX_PREFIXES 1024

/*
 * Routed decode step behind shared prefixes: swattn_decode_fwd where the keys of sequence
 * b are the first prefix_lens[i] rows of prefix i = prefix_ids[b], then the first
 * cache_lens[b] rows of its own cache.  With n of them together the new token sits at
 * position n - 1 and attends all n where full[b], else the last `window` of them.  A
 * prefix's rows are read once for every 128 query rows of a KV head that attend them (of
 * G = heads_q / heads_kv for each sequence), full and local routes apart.
 *
 *   q                   bf16 [batch, heads_q, 128]
 *   k_prefix, v_prefix  bf16 [prefixes, prefix_len, heads_kv, 128]
 *   prefix_lens         int32 [prefixes], clamped to [0, prefix_len]
 *   prefix_ids          int32 [batch]; a sequence whose id lies outside [0, prefixes) has
 *                       no prefix
 *   k_cache, v_cache    bf16 [batch, cache_len, heads_kv, 128]
 *   cache_lens          int32 [batch], clamped to [0, cache_len]; own rows, the new token's
 *                       among them
 *   full                uint8 [batch]
 *   out, lse            bf16 [batch, heads_q, 128], fp32 [batch, heads_q] (log2); a sequence
 *                       without keys gets O = NaN, LSE = -inf
 *   workspace           >= swattn_shared_decode_workspace_bytes(), asked on the current
 *                       device; 256-byte aligned
 * heads_q / heads_kv at most 8; batch up to SWATTN_SHARED_MAX_SEQS, prefixes 1 to
 * SWATTN_SHARED_MAX_PREFIXES; below 2^31 both batch * heads_kv * (cache_len + 192) and
 * tiles * heads_kv * (prefix_len + 64), with tiles = min(batch, 2 * prefixes + batch /
 * (128 / G)), divisions rounded down; batch * heads_q below 2^24.  The workspace query
 * returns 0 for shapes that are refused.  scale_log2 is finite.
 */
size_t swattn_shared_decode_workspace_bytes(int32_t batch, int64_t cache_len, int32_t prefixes,
                                            int64_t prefix_len, int32_t heads_q,
                                            int32_t heads_kv);
int swattn_shared_decode_fwd(const void* q, const void* k_prefix, const void* v_prefix,
                             const int32_t* prefix_lens, const int32_t* prefix_ids,
                             const void* k_cache, const void* v_cache, const int32_t* cache_lens,
                             const uint8_t* full, void* out, float* lse, int32_t batch,
                             int64_t cache_len, int32_t prefixes, int64_t prefix_len,
                             int32_t heads_q, int32_t heads_kv, int32_t head_dim, int32_t window,
                             float scale_log2, void* workspace, size_t workspace_bytes,
                             void* stream);

#ifdef __cplusplus
}  // extern "C"
#endif

#endif  // SWATTN_SHARED_H_
