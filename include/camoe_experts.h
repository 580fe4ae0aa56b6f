/*
 * camoe_experts.h — C ABI of the expert layer that follows the time mix in
 * CaMoE (the reference sends each token to its top-2 experts by boolean masks,
 * camoe/system.py:263-297, and each RWKV expert is a squared-ReLU feed-forward
 * product, camoe/experts.py), and of a projection with low-rank adapters.
 *
 * N tokens of width C choose k experts each; slot s = n k + j is token n's
 * j-th choice.  A slot whose expert is outside [0, E) is unused (dropped by a
 * capacity limit, padding): it reads nothing and contributes nothing.  The R =
 * N k rows of the sorted arrays hold the used slots in the order of their
 * experts, slots of one expert in their own order (a stable sort), and zeros
 * behind them:
 *
 *   offsets [E + 1]  expert e owns rows [offsets[e], offsets[e + 1])
 *   position [N, k]  the row of each slot, -1 for an unused one
 *   source [R]       the slot of each row, -1 behind offsets[E]
 *
 * All three are int32, so R is at most 2^31 - 1.  dtype is 0 (bf16) or 1
 * (fp32); arithmetic is fp32.  All arrays are contiguous; those of the products
 * and adapters are 16-byte aligned, those of the sort, the copies and the sums
 * need their element's alignment (and are fastest at 16 bytes); other addresses
 * are refused.  Calls are
 * asynchronous on `stream`, allocate nothing, and return the status codes of
 * camoe_wkv7.h (0 = ok).  1 <= E <= 1024, 1 <= k <= 64.
 */
#ifndef CAMOE_EXPERTS_H
#define CAMOE_EXPERTS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace of camoe_ex_dispatch (may be 0, then work may be NULL). */
size_t camoe_ex_dispatch_work_bytes(int64_t N, int64_t k, int64_t E);

/* Sort the slots and copy the tokens: index [N, k] holds the chosen experts
 * (index_bytes 4: int32, 8: int64), xs[p] = x[source[p] / k], zeros in the rows
 * behind offsets[E].  xs NULL (then x may be NULL too) sorts only. */
int camoe_ex_dispatch(const void* x, int dtype, const void* index, int index_bytes, void* xs,
                      int32_t* offsets, int32_t* position, int32_t* source, void* work,
                      size_t work_bytes, int64_t N, int64_t k, int64_t E, int64_t C, void* stream);

/* out[n] = sum over j of weight[n, j] rows[position[n, j]] (fp32 weight; NULL
 * means ones), rounded once: the experts' rows back to their tokens, and the
 * gradient of camoe_ex_dispatch.  A token without a used slot gets zeros. */
int camoe_ex_combine(const void* rows, int dtype, const float* weight, const int32_t* position,
                     void* out, int64_t N, int64_t k, int64_t C, void* stream);

/* Backward of camoe_ex_combine with weights: dys[p] = weight[source[p]]
 * dout[source[p] / k], zeros behind offsets[E]; dweight[n, j] = <dout[n],
 * ys[position[n, j]]>, 0 for an unused slot.  dys or dweight may be NULL. */
int camoe_ex_combine_bwd(const void* dout, int dtype, const void* ys, const float* weight,
                         const int32_t* offsets, const int32_t* position, void* dys,
                         float* dweight, int64_t N, int64_t k, int64_t E, int64_t C, void* stream);

/* The experts' products over sorted rows, bf16: for the rows p of expert e
 *   h[p]  = relu(w_up[e] xs[p])^2      w_up   [E, F, C]
 *   ys[p] = w_down[e] h[p]             w_down [E, C, F]
 * h [R, F] is written too, and h_low [R, F rounded up to 16] (bytes, may be
 * NULL): the 8 bits of h below bf16's, for the backward.  The rows behind offsets[E] of ys are zeros.
 * C and F are multiples of 8. */
int camoe_ex_ffn_fwd(const void* xs, const void* w_up, const void* w_down, const int32_t* offsets,
                     void* h, void* h_low, void* ys, int64_t R, int64_t E, int64_t C, int64_t F, void* stream);

/* Backward of camoe_ex_ffn_fwd: dpre [R, F] is scratch; dxs [R, C], dw_up
 * [E, F, C] and dw_down [E, C, F] are bf16 and each may be NULL.  h and h_low
 * are the forward's (h_low may be NULL: h as rounded to bf16 is used alone).  An
 * expert without rows gets zero weight gradients. */
int camoe_ex_ffn_bwd(const void* dys, const void* xs, const void* w_up, const void* w_down,
                     const int32_t* offsets, const void* h, const void* h_low, void* dpre, void* dxs,
                     void* dw_up, void* dw_down, int64_t R, int64_t E, int64_t C, int64_t F, void* stream);

/* Bytes of workspace of camoe_ad_linear. */
size_t camoe_ad_work_bytes(int64_t N, int64_t C, int64_t M, int64_t D, int64_t L);

/* A projection shared by all rows with the adapter of each row beside it, bf16:
 *   y[n] = weight x[n] + scale[a] up[a] (down[a] x[n]),   a = adapter[n]
 * weight [M, C], down [L, D, C], up [L, M, D], scale [L] fp32 (NULL: ones),
 * adapter [N] int32; a row whose adapter is outside [0, L) gets weight x[n]
 * alone.  C, M and D are multiples of 8, D <= 256, L <= 1024.  y is rounded once;
 * with many rows (above 128, or above 512 where N M D <= 24 * 2^20) scale down x is
 * rounded to bf16 before its product with up.  Values of an adapter that are not
 * finite reach its own rows only. */
int camoe_ad_linear(const void* x, const void* weight, const void* down, const void* up,
                    const int32_t* adapter, const float* scale, void* y, void* work,
                    size_t work_bytes, int64_t N, int64_t C, int64_t M, int64_t D, int64_t L,
                    void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CAMOE_EXPERTS_H */
