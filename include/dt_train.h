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
 * The norm of every query and key head with the rotate-half RoPE in the same pass:
 *   y = x * rsqrt(mean(x^2) + eps) * w          x a head of q or k, w = w_q or w_k [D]
 *   out[i] = y[i] cos[t, i] - y[i + D/2] sin[t, i],
 *   out[i + D/2] = y[i + D/2] cos[t, i + D/2] + y[i] sin[t, i + D/2]        i < D/2
 * at table row t = start_pos[b] + s (start_pos null: s).  q, q_out [B, S, Hq, D], k,
 * k_out [B, S, Hkv, D], D contiguous; strides holds the (batch, position, head)
 * element strides of q, k, q_out and k_out, 12 values.  Any head numbers; even D from 2
 * to 256, bf16, fp16 or fp32, any strides and alignment (D a multiple of 16, or of 8 in
 * fp32, with 16-byte aligned heads and table rows runs fastest; 16-bit heads of a multiple
 * of 8 on 8-byte boundaries come next).
 * Weights in the same type, or in fp32 with weights_fp32.  cos / sin [cos_rows, D] fp32
 * with a common row stride.  A position outside the tables sets the device status word
 * and its outputs to zeros.  An output may be its own input.  fp32 arithmetic, one
 * rounding.
 */
int dt_head_norm_rope_forward(const void* q, const void* k, const void* w_q, const void* w_k, void* q_out, void* k_out,
                              const float* cos_tab, const float* sin_tab, int64_t cos_stride, int cos_rows,
                              const int32_t* start_pos, int B, int S, int Hq, int Hkv, int D, const int64_t* strides,
                              int weights_fp32, float eps, int dtype, void* stream);

/* Bytes of scratch that dt_head_norm_rope_backward needs on the current device;
 * negative on an error. */
int64_t dt_head_norm_rope_workspace(int B, int S, int Hq, int Hkv, int D);

/*
 * Gradient of dt_head_norm_rope_forward from dq_out and dk_out: dq, dk (which may be
 * dq_out and dk_out themselves), dw_q, dw_k [D] in the weights' type.  strides: of q,
 * k, dq, dk, dq_out and dk_out, 18 values.  workspace: dt_head_norm_rope_workspace
 * bytes, 16-byte aligned.  Deterministic: sums are fp32 and in a fixed order.
 */
int dt_head_norm_rope_backward(const void* dq_out, const void* dk_out, const void* q, const void* k, const void* w_q,
                               const void* w_k, void* dq, void* dk, void* dw_q, void* dw_k, const float* cos_tab,
                               const float* sin_tab, int64_t cos_stride, int cos_rows, const int32_t* start_pos,
                               void* workspace, int64_t workspace_bytes, int B, int S, int Hq, int Hkv, int D,
                               const int64_t* strides, int weights_fp32, float eps, int dtype, void* stream);

/*
 * y = residual + dropout(x) (residual null: 0) over rows [rows, cols]; the
 * gradient of x is the same call on the gradient of y without a residual.
 * bf16, fp16 or fp32, 1 <= cols <= 2^31 - 256, any strides and alignment
 * (contiguous 16-byte aligned rows of a multiple of 8 elements run faster); y
 * overlaps neither input.
 */
int dt_dropout(const void* x, int64_t x_stride, const void* residual, int64_t res_stride, void* y, int64_t y_stride,
               int64_t rows, int cols, double p, const int64_t* rng, uint32_t site, int dtype, void* stream);

/*
 * The 2-norm of many tensors taken as one: norm (fp32, one number) receives
 * sqrt(sum of squares).  tensors: their addresses (0: left out), sizes: numbers of
 * elements (whole tensors without gaps, any order of dimensions), kinds: dtype codes.
 * Any alignment.  The three arrays are the host's and are read during the call.  Pairs
 * of squares are added in fp32, the rest in fp64 (all of it where fp32 would overflow or
 * lose bits), in a fixed order.  workspace: dt_grad_norm_workspace bytes, 16-byte aligned.
 */
int dt_grad_norm(int count, const int64_t* tensors, const int64_t* sizes, const int32_t* kinds, float* norm,
                 void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of scratch that dt_grad_norm and the clipping of dt_adamw_step need for `count`
 * tensors on the current device; negative on an error. */
int64_t dt_grad_norm_workspace(int count);

/* Hyperparameters of a group of tensors: betas in [0, 1), eps a normal fp32 number, the
 * others not negative.  lr_tensor: the rate as an fp32 number on the device, read by the
 * kernel, or null: lr. */
typedef struct {
  double lr, beta1, beta2, eps, weight_decay;
  const float* lr_tensor;
} DtAdamWGroup;

/*
 * One AdamW step over many tensors:
 *   g' = g min(1, max_norm / (norm + 1e-6))      norm: of all gradients; max_norm <= 0: g' = g
 *   m' = beta1 m + (1 - beta1) g',  v' = beta2 v + (1 - beta2) g'^2
 *   p' = p (1 - lr weight_decay) - lr / (1 - beta1^t) m' / (sqrt(v') / sqrt(1 - beta2^t) + eps)
 * params, grads: addresses of weights and gradients (gradient 0: the tensor is left alone),
 * of the same dtype, size and order of elements, whole tensors without gaps, any
 * alignment; sizes: numbers of elements; kinds: dtype code + 256 * group.  1 to 16 groups.
 * The arrays are the host's and are read during the call.
 *
 * The averages are flat arrays: tensor i's begin at 256 times the number of blocks of 256
 * elements of the tensors before it (the last block of each filled up), 16-byte aligned.
 * state_bits 32: fp32.  state_bits 8: one byte an element and one for each block of 256,
 * the biased exponent e (32 at least) of the block's largest value; exp_avg as sign, four
 * exponent and three further bits (a number of type e4m3) times 2^(e - 134), exp_avg_sq as
 * five exponent and three further bits (those of a half number under its sign) times
 * 2^(e - 141).  They are rounded up or down at random: element i of the flat array goes up
 * when the part cut off and w / 2^16 come to a step, w word i % 8 of the generator's block
 * i / 8 (above; site 2^32 - 1, step t), for exp_avg with its two bytes turned over.  An
 * exp_avg_sq above zero is never stored as zero.  A block with a value that is not finite
 * reads as NaN from then on (e = 255).
 *
 * master: fp32 weights of the 16-bit tensors, flat in the same way, or null: then p' is
 * computed from the weight itself and rounded.  state: (seed, steps taken), 64-bit
 * integers; t = steps taken + 1, which the call counts.  ticket: a zero that the call
 * leaves as one.  With max_norm the norm is written to `norm`, and where it is not finite
 * nothing else is written and the step is not counted; workspace as dt_grad_norm's.
 * Deterministic.  Arithmetic in fp32, the steps' powers in fp64.
 */
int dt_adamw_step(int count, const int64_t* params, const int64_t* grads, const int64_t* sizes, const int32_t* kinds,
                  int ngroups, const DtAdamWGroup* groups, int state_bits, void* exp_avg, void* exp_avg_sq,
                  uint8_t* exp_avg_scale, uint8_t* exp_avg_sq_scale, float* master, int64_t* state, uint32_t* ticket,
                  double max_norm, float* norm, void* workspace, int64_t workspace_bytes, void* stream);

/* The numbers that 8-bit averages stand for, as bf16 (which holds each of them): [256 * blocks] each. */
int dt_adamw_moments(const uint8_t* exp_avg, const uint8_t* exp_avg_scale, const uint8_t* exp_avg_sq,
                     const uint8_t* exp_avg_sq_scale, int64_t blocks, void* exp_avg_out, void* exp_avg_sq_out,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DT_TRAIN_H_ */
