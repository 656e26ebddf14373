/*
 * dt_train.h -- C ABI of the training operators of libdt_attn_sm100.so: the
 * parts of a Decision Transformer block's training step that are not plain
 * matrix products, forward and backward.
 *
 * Conventions are those of dt_attn.h: raw device pointers, sizes, element
 * strides, a cudaStream_t passed as void*, status codes with dt_last_error();
 * no entry point allocates device memory or waits for the device.  Calls that
 * need scratch take it from the caller.
 *
 * Dropout masks are never stored.  `rng` points at two 64-bit integers on the
 * device, (seed, step), read by the kernels; with the call's `site` number they
 * key Philox4x32 with seven rounds: counter (block low, block high, step low
 * word, site), key = seed, eight 16-bit words a block (low half of output word
 * 0 first).  Element (row, col) of a tensor of rows of n elements uses word
 * col % 8 of block row * ceil(n / 8) + col / 8, and stays iff that word is >=
 * round(p * 65536); survivors are scaled by 65536 / (65536 - round(p * 65536)).
 * A dropped element contributes 0 whatever its value.  The backward call gives
 * the same rng contents, site and p as the forward call.  With p = 0 rng may be
 * null.  p must lie in [0, 1) and round(p * 65536) below 65536.
 */
#ifndef DT_TRAIN_H_
#define DT_TRAIN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Causal grouped-query attention with dropout on the attention weights, for
 * training.  q, o [B, S, Hq, D]; k, v [B, S, Hkv, D] (already rotated q and k;
 * element strides, D contiguous, 16-byte aligned pointers, strides multiples
 * of 8); bf16 or fp16; D in {32, 64}; Hq a multiple of Hkv; S >= 1.
 * pad_len [B] (or null) counts leading padding positions: keys and queries
 * below it take no part; their output rows are zeros (dt_attn_prefill, the
 * inference form, gives such rows the reference's mean of V instead) and
 * nothing of theirs is read.  scale <= 0 means 1 / sqrt(D).  The dropout row of
 * query s of head h of sample b is (b * Hq + h) * S + s, its columns the keys.
 * lse [B, Hq, S] fp32 receives the base-2 logarithm of each row's softmax
 * denominator (+inf for a row without keys), the backward call's input.
 * workspace: dt_attn_train_forward_workspace bytes, 16-byte aligned.  Values that
 * are not finite never leave padding, their sample or their KV head.  Within those,
 * a zero weight times them is not a zero: in k and v they may reach rows of o (and
 * dq) up to 190 positions before them, in q and dout the dk and dv of keys up to
 * 127 positions behind them.
 */
int dt_attn_train_forward(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* pad_len,
                          int B, int S, int Hq, int Hkv, int D, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                          int64_t k_sb, int64_t k_ss, int64_t k_sh, int64_t v_sb, int64_t v_ss, int64_t v_sh,
                          int64_t o_sb, int64_t o_ss, int64_t o_sh, void* workspace, int64_t workspace_bytes,
                          float scale, double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

/* Bytes of scratch that dt_attn_train_forward needs on the current device: 0 (then
 * workspace may be null) unless rows are too few for the GPU and the walk over
 * their keys is cut; negative on an error. */
int64_t dt_attn_train_forward_workspace(int B, int S, int Hq, int Hkv, int D);

/*
 * Gradient of dt_attn_train_forward: dq [B, S, Hq, D], dk, dv [B, S, Hkv, D]
 * (summed over the query heads that share a KV head) from dout and the forward
 * call's inputs, o and lse.  strides holds the (batch, position, head) strides
 * of q, k, v, o, dout, dq, dk and dv in that order, 24 values.  workspace:
 * dt_attn_train_workspace bytes, 16-byte aligned.  Deterministic: every sum is
 * taken in a fixed order.
 */
int dt_attn_train_backward(const void* dout, const void* q, const void* k, const void* v, const void* o,
                           const float* lse, void* dq, void* dk, void* dv, const int32_t* pad_len, void* workspace,
                           int64_t workspace_bytes, int B, int S, int Hq, int Hkv, int D, const int64_t* strides,
                           float scale, double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

/* Bytes of scratch that dt_attn_train_backward needs on the current device (more
 * with has_dropout, the p > 0 of its call, than without); negative on an error. */
int64_t dt_attn_train_workspace(int B, int S, int Hq, int Hkv, int D, int has_dropout);

/*
 * Gradient of the RoPE that dt_qkv_rope applies to the q and k heads, in place
 * on the gradient of its output: columns [0, rope_cols) of g [rows, N] (row
 * stride in elements), groups of head_dim (32 or 64), row r rotated back by
 * table row (r mod seq_len) of cos / sin ([>= seq_len, head_dim] fp32).  bf16 or
 * fp16; stride and rope_cols multiples of 8 and head_dim, g 16-byte and cos /
 * sin 8-byte aligned with an even row stride.
 */
int dt_rope_grad(void* g, int64_t g_stride, int64_t rows, const float* cos_tab, const float* sin_tab,
                 int64_t cos_stride, int cos_rows, int seq_len, int rope_cols, int head_dim, int dtype, void* stream);

/*
 * Residual add with the norms before and after it, a gate and dropout:
 *   u = x * rsqrt(mean(x^2) + eps) * w_post    (u = x when w_post is null)
 *   h = residual + alpha * gate * dropout(u)   (residual null: 0; gate null: 1)
 *   n = h * rsqrt(mean(h^2) + eps) * w_pre
 * x, residual, h, n [M, H] (h and n without gaps between rows), w_pre, w_post
 * [H], gate [M / gate_rows, H]: gate_rows consecutive rows share a row of it.
 * bf16, fp16 or fp32 throughout; 1 <= H <= 8192, any strides and alignment (16-byte
 * aligned rows of a multiple of 8 elements run faster).  Arithmetic in fp32,
 * each output rounded once, n from the unrounded h.  stats [M, 2] fp32 receives
 * the two reciprocal roots for the backward call.
 */
int dt_residual_norm_forward(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
                             const void* gate, int64_t gate_stride, int64_t gate_rows, const void* w_pre,
                             const void* w_post, void* h, void* n, float* stats, int64_t M, int H, float alpha,
                             float eps, double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

/* Bytes of scratch that dt_residual_norm_backward needs on the current device
 * (gate_rows 0: no gate); negative on an error. */
int64_t dt_residual_norm_workspace(int64_t M, int H, int64_t gate_rows, int has_post);

/*
 * Gradient of dt_residual_norm_forward from dh (of h, nullable: zero) and dn
 * (of n, nullable: zero; not both null): dx and dresidual [M, H] without gaps
 * (dresidual nullable), dw_pre [H] (zeros are not written: null when dn is
 * null), dw_post [H] (with w_post), dgate [M / gate_rows, H] (with gate).
 * workspace: dt_residual_norm_workspace bytes, 16-byte aligned.  Deterministic.
 */
int dt_residual_norm_backward(const void* dh, int64_t dh_stride, const void* dn, int64_t dn_stride, const void* x,
                              int64_t x_stride, const void* residual, int64_t res_stride, const void* gate,
                              int64_t gate_stride, int64_t gate_rows, const void* w_pre, const void* w_post,
                              const float* stats, void* dx, void* dresidual, void* dw_pre, void* dw_post, void* dgate,
                              void* workspace, int64_t workspace_bytes, int64_t M, int H, float alpha, float eps,
                              double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

/*
 * y = residual + dropout(x) (residual null: 0) over rows [rows, cols]; the
 * gradient of x is the same call on the gradient of y without a residual.
 * bf16, fp16 or fp32, 1 <= cols <= 2^31 - 256, any strides and alignment
 * (contiguous 16-byte aligned rows of a multiple of 8 elements run faster); y
 * overlaps neither input.
 */
int dt_dropout(const void* x, int64_t x_stride, const void* residual, int64_t res_stride, void* y, int64_t y_stride,
               int64_t rows, int cols, double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DT_TRAIN_H_ */
