/*
 * swattn_rotary.h -- C ABI of libswattn.so for what stands between a layer's
 * projections and its attention: the norm of every query and key head and the
 * rotation by positions in one pass, forward and backward, and the same with the
 * keys (and values) written into bf16 caches.  The conventions are those of
 * swattn.h: device pointers unless marked "host", a hipStream_t passed as void*, no
 * allocation, no synchronisation, the same status codes and swattn_last_error().
 * Nothing here has a counterpart in the reference, which starts at finished Q and K.
 *
 * A head row x of 128 dims becomes
 *   y = w x / sqrt(mean(x^2) + eps)      (weight NULL: y = x)
 *   (a, b) -> (a cos t - b sin t, b cos t + a sin t)
 * for the first `rotary` dims, rotary = 2 * (number of frequencies), a multiple of 16
 * up to 128.  Pair i of them is (y[i], y[i + rotary / 2]), or (y[2 i], y[2 i + 1]) with
 * `interleaved`; its angle t is inv_freq[i] times the token's position on the axis that
 * frequency i belongs to.  Dims from `rotary` on stay as they are.
 *
 * Shared arguments:
 *   q, k          bf16 rows, element (b, s, h, d) at b * strides[0] + s * strides[1] + h *
 *                 strides[2] + d (host arrays of 3): slices of a fused projection are
 *                 taken as they are.  Strides are not negative and multiples of 8, the
 *                 base 16-byte aligned.
 *   positions     int32 [axes, batch, seq], any sign
 *   inv_freq      fp32 (freq_f64 0) or fp64 (freq_f64 1) [rotary / 2], below 2^40 in
 *                 magnitude; angles are its values times the positions, off by at most
 *                 2^-65 turns per position (2^-34 turns at the ends of int32), and their
 *                 sines and cosines by 8 roundings of fp32 of themselves beside that.
 *                 Others, NaN among them, give NaN.
 *   sections      host int32 [axes]: how many of the frequencies, in order, belong to
 *                 each axis; positive, their sum is the number of frequencies.  axes 1 to 4
 *   q_weight, k_weight  fp32 (weight_bf16 0) or bf16 (1) [128], or NULL: not normalised
 */
#ifndef SWATTN_ROTARY_H_
#define SWATTN_ROTARY_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SWATTN_ROTARY_MAX_AXES 4

/*
 * Rotate: q_out [batch, seq, heads_q, 128] and k_out [batch, seq, heads_kv, 128], bf16,
 * contiguous.  They may not overlap the inputs.
 */
int swattn_rotary_fwd(const void* q, const int64_t* q_strides, const void* k,
                      const int64_t* k_strides, const int32_t* positions, const void* inv_freq,
                      int32_t freq_f64, const int32_t* sections, int32_t axes,
                      int32_t interleaved, const void* q_weight, const void* k_weight,
                      int32_t weight_bf16, float eps, void* q_out, void* k_out, int32_t batch,
                      int64_t seq, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                      void* stream);

/*
 * Gradients of swattn_rotary_fwd's outputs: grad_q, grad_k as its outputs, q and k as its
 * inputs (looked at only where the tensor has a weight, else NULL will do); dq and dk like
 * the outputs.
 *   dq_weight, dk_weight  [128] of the weights' type, or NULL: not wanted (always NULL
 *                         where there is no weight).  Summed in fp32 in a fixed order.
 *   workspace   >= swattn_rotary_bwd_workspace_bytes(), asked on the current device;
 *               256-byte aligned.  Not looked at where no weight's gradient is wanted.
 */
size_t swattn_rotary_bwd_workspace_bytes(int32_t batch, int64_t seq, int32_t heads_q,
                                         int32_t heads_kv);
int swattn_rotary_bwd(const void* grad_q, const void* grad_k, const void* q,
                      const int64_t* q_strides, const void* k, const int64_t* k_strides,
                      const int32_t* positions, const void* inv_freq, int32_t freq_f64,
                      const int32_t* sections, int32_t axes, int32_t interleaved,
                      const void* q_weight, const void* k_weight, int32_t weight_bf16, float eps,
                      void* dq, void* dk, void* dq_weight, void* dk_weight, int32_t batch,
                      int64_t seq, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * Rotate q to q_out, and k into rows cache_lens[b] .. of a bf16 cache [batch, cache_len,
 * heads_kv, 128], v (strides as q's) into the same rows of another, unchanged.
 *   cache_lens  int32 [batch]: valid rows before the call, clamped to [0, cache_len]
 *   counts      int32 [batch], clamped to [0, seq], or NULL: tokens that each sequence
 *               appends (NULL: all); the q rows of the others are rotated like the rest
 *   lens_out    int32 [batch]: min(cache_lens + counts, cache_len).  May not alias cache_lens.
 * Rows that would lie behind cache_len are dropped.
 */
int swattn_rotary_append(const void* q, const int64_t* q_strides, const void* k,
                         const int64_t* k_strides, const void* v, const int64_t* v_strides,
                         const int32_t* positions, const void* inv_freq, int32_t freq_f64,
                         const int32_t* sections, int32_t axes, int32_t interleaved,
                         const void* q_weight, const void* k_weight, int32_t weight_bf16, float eps,
                         void* q_out, void* k_cache, void* v_cache, const int32_t* cache_lens,
                         const int32_t* counts, int32_t* lens_out, int32_t batch, int64_t seq,
                         int64_t cache_len, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                         void* stream);

#ifdef __cplusplus
}  // extern "C"
#endif

#endif  // SWATTN_ROTARY_H_
