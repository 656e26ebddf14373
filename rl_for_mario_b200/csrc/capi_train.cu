// C-ABI entry points of the training operators (include/dt_train.h): argument
// validation and dispatch.  No entry point allocates device memory.
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cmath>
#include <initializer_list>

#include "../../include/dt_attn.h"
#include "../../include/dt_train.h"
#include "dt_internal.h"

namespace {

using dtk::api_fail;

struct Range {
  explicit Range(const char* name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
  Range(const Range&) = delete;
  Range& operator=(const Range&) = delete;
};

int cuda_status(cudaError_t e, const char* what) {
  return e == cudaSuccess ? DT_OK : api_fail(DT_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int need_sm100(const char* fn, int* num_sms, int** status_out = nullptr) {
  int* status = nullptr;
  int cc = 0;
  const int rc = dtk::api_device(&status, &cc, num_sms);
  if (rc) return rc;
  if (status_out) *status_out = status;
  if (cc != 10) return api_fail(DT_ERR_UNSUPPORTED, "%s: needs an sm_100 GPU (current device is cc %d.x)", fn, cc);
  return DT_OK;
}

// The dropout rate as the kernels use it: p in units of 2^-16.
int rate(const char* fn, double p, const int64_t* rng, uint32_t* threshold, float* inv_keep) {
  if (!(p >= 0.0 && p < 1.0)) return api_fail(DT_ERR_INVALID, "%s: p must lie in [0, 1) (got %g)", fn, p);
  const double t = nearbyint(p * 65536.0);
  if (t >= 65536.0) return api_fail(DT_ERR_INVALID, "%s: p = %.9g rounds to 1 in units of 2^-16", fn, p);
  *threshold = (uint32_t)t;
  *inv_keep = (float)(65536.0 / (65536.0 - t));
  if (*threshold && !rng) return api_fail(DT_ERR_INVALID, "%s: null rng with p > 0", fn);
  if (reinterpret_cast<uintptr_t>(rng) & 7) return api_fail(DT_ERR_INVALID, "%s: rng must be 8-byte aligned", fn);
  return DT_OK;
}

int elem_size(int dtype) { return dtype == DT_DTYPE_FP32 ? 4 : 2; }

int check_dtype(const char* fn, int dtype) {
  if (dtype != DT_DTYPE_BF16 && dtype != DT_DTYPE_FP16 && dtype != DT_DTYPE_FP32)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
  return DT_OK;
}

int check_attn(const char* fn, int B, int S, int Hq, int Hkv, int D, const int64_t* strides, int nstrides, int dtype) {
  if (B < 1 || S < 1 || Hq < 1 || Hkv < 1)
    return api_fail(DT_ERR_INVALID, "%s: sizes must be positive (B=%d S=%d Hq=%d Hkv=%d)", fn, B, S, Hq, Hkv);
  if (Hq % Hkv != 0)
    return api_fail(DT_ERR_INVALID, "%s: num_attention_heads (%d) must be divisible by num_key_value_heads (%d)", fn,
                    Hq, Hkv);
  if (D != 32 && D != 64) return api_fail(DT_ERR_UNSUPPORTED, "%s: head_dim %d not in {32, 64}", fn, D);
  if (dtype != DT_DTYPE_BF16 && dtype != DT_DTYPE_FP16)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16 or fp16)", fn, dtype);
  for (int i = 0; i < nstrides; ++i)
    if (strides[i] <= 0 || strides[i] % 8 != 0)
      return api_fail(DT_ERR_INVALID, "%s: stride #%d (%lld) must be a positive multiple of 8", fn, i,
                      (long long)strides[i]);
  if ((long long)((S + 63) / 64) * B * Hq > 0x3fffffffLL)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: too many query tiles (B=%d S=%d Hq=%d)", fn, B, S, Hq);
  return DT_OK;
}

int check_rows(const char* fn, const void* x, int64_t M, int H, const char* m_name, const char* h_name) {
  if (!x) return api_fail(DT_ERR_INVALID, "%s: null x", fn);
  if (M < 1 || H < 1)
    return api_fail(DT_ERR_INVALID, "%s: sizes must be positive (%s=%lld %s=%d)", fn, m_name, (long long)M, h_name, H);
  return DT_OK;
}

// Rows wide enough not to overlap is the caller's business for inputs; element
// alignment is checked, as every access relies on it.
int check_elem_aligned(const char* fn, int dtype, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % elem_size(dtype))
      return api_fail(DT_ERR_INVALID, "%s: a pointer is not aligned to its elements", fn);
  return DT_OK;
}

// The backward pass's scratch: delta, then the partial sums of split tiles, then the drop flags, then (fp16) the
// parts of the gradients' scale.
int64_t delta_elems(int B, int S, int Hq) { return ((int64_t)B * Hq * S + 3) / 4 * 4; }
int64_t attn_row_part_elems(int B, int S, int Hq, int Hkv, int D, int sms) {
  const int n = dtk::attn_train_row_splits(B, S, Hkv, Hq / Hkv, sms);
  return n > 1 ? (int64_t)n * B * Hq * S * D : 0;
}
int64_t attn_part_elems(int B, int S, int Hq, int Hkv, int D, int sms) {  // dq's are read before dk's and dv's come
  const int n = dtk::attn_train_splits(B, S, Hkv, Hq / Hkv, sms);
  const int64_t keys = n > 1 ? (int64_t)n * 2 * B * Hkv * S * D : 0, rows = attn_row_part_elems(B, S, Hq, Hkv, D, sms);
  return keys > rows ? keys : rows;
}
int64_t attn_forward_workspace(int B, int S, int Hq, int Hkv, int D, int sms) {
  return attn_row_part_elems(B, S, Hq, Hkv, D, sms) / D * (D + 2) * 4;
}
int64_t attn_workspace(int B, int S, int Hq, int Hkv, int D, bool drop, int sms) {
  return 4 * (delta_elems(B, S, Hq) + attn_part_elems(B, S, Hq, Hkv, D, sms) +
              (drop ? dtk::attn_train_words(B, S, Hq, D) : 0) +
              (int64_t)B * Hkv * dtk::attn_train_grad_parts(S, Hq / Hkv, D) * 2);
}

constexpr int kMaxCols = 0x7fffff00;  // of dropout: columns are numbered in 32 bits, in pieces of 256
constexpr int kMaxHidden = 8192;  // 32 warps of 256 columns: one block holds a row

int64_t part_elems(const dtk::ResidualNormPlan& q, int H, int64_t gate_rows, bool post) {
  int64_t n = 0;
  if (q.grid > 1) n += q.grid * (post ? 2 : 1);
  if (gate_rows > 1 && q.chunks_per_span > 1) n += q.chunks;
  // Each part starts on a 16-byte boundary: rows of H floats, H rounded up.
  return n * ((H + 3) / 4 * 4) + 16;
}

}  // namespace

extern "C" {

int dt_attn_train_forward(const void* q, const void* k, const void* v, void* o, float* lse, const int32_t* pad_len,
                          int B, int S, int Hq, int Hkv, int D, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                          int64_t k_sb, int64_t k_ss, int64_t k_sh, int64_t v_sb, int64_t v_ss, int64_t v_sh,
                          int64_t o_sb, int64_t o_ss, int64_t o_sh, void* workspace, int64_t workspace_bytes,
                          float scale, double p, const int64_t* rng, uint32_t site, int dtype, void* stream) {
  const char* fn = "dt_attn_train_forward";
  Range range(fn);
  if (!q || !k || !v || !o || !lse) return api_fail(DT_ERR_INVALID, "%s: null q/k/v/o/lse pointer", fn);
  const int64_t strides[12] = {q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh};
  int rc = check_attn(fn, B, S, Hq, Hkv, D, strides, 12, dtype);
  if (rc) return rc;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return api_fail(DT_ERR_INVALID, "%s: q/k/v/o must be 16-byte aligned", fn);
  dtk::AttnTrainParams a{};
  if ((rc = rate(fn, p, rng, &a.threshold, &a.inv_keep))) return rc;
  int sms = 0;
  if ((rc = need_sm100(fn, &sms, &a.status))) return rc;
  const int64_t need = attn_forward_workspace(B, S, Hq, Hkv, D, sms);
  if (need && (workspace_bytes < need || !workspace || !aligned16(workspace)))
    return api_fail(DT_ERR_INVALID, "%s: workspace of %lld bytes is too small, null or not 16-byte aligned", fn,
                    (long long)workspace_bytes);
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + attn_row_part_elems(B, S, Hq, Hkv, D, sms);
  a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse, a.pad_len = pad_len;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.k_sb = k_sb, a.k_ss = k_ss, a.k_sh = k_sh;
  a.v_sb = v_sb, a.v_ss = v_ss, a.v_sh = v_sh, a.o_sb = o_sb, a.o_ss = o_ss, a.o_sh = o_sh;
  a.B = B, a.S = S, a.Hq = Hq, a.Hkv = Hkv, a.R = Hq / Hkv;
  a.scale = scale > 0.f ? scale : 1.0f / sqrtf((float)D);
  a.rng = reinterpret_cast<const long long*>(rng);
  a.site = site;
  a.HC = a.R < 64 ? a.R : 64;
  a.PT128 = 128 / a.HC, a.PT64 = 64 / a.HC, a.by_pt64 = dtk::FastDiv((uint32_t)a.PT64);
  const bool bf16 = dtype == DT_DTYPE_BF16;
  dtk::AttnTrainMaps m;
  if ((rc = dtk::api_encode_bshd(&m.q_tile, q, bf16, B, S, Hq, D, q_sb, q_ss, q_sh, a.HC, 128 / a.HC, "q")) ||
      (rc = dtk::api_encode_bshd(&m.k_blk, k, bf16, B, S, Hkv, D, k_sb, k_ss, k_sh, 1, 64, "k")) ||
      (rc = dtk::api_encode_bshd(&m.v_blk, v, bf16, B, S, Hkv, D, v_sb, v_ss, v_sh, 1, 64, "v")))
    return rc;
  return cuda_status(dtk::launch_attn_train_fwd_sm100(a, m, D, bf16, sms, static_cast<cudaStream_t>(stream)), fn);
}

int dt_attn_train_backward(const void* dout, const void* q, const void* k, const void* v, const void* o,
                           const float* lse, void* dq, void* dk, void* dv, const int32_t* pad_len, void* workspace,
                           int64_t workspace_bytes, int B, int S, int Hq, int Hkv, int D, const int64_t* strides,
                           float scale, double p, const int64_t* rng, uint32_t site, int dtype, void* stream) {
  const char* fn = "dt_attn_train_backward";
  Range range(fn);
  if (!dout || !q || !k || !v || !o || !lse || !workspace || !dq || !dk || !dv || !strides)
    return api_fail(DT_ERR_INVALID, "%s: null pointer", fn);
  int rc = check_attn(fn, B, S, Hq, Hkv, D, strides, 24, dtype);
  if (rc) return rc;
  for (const void* t : {dout, q, k, v, o, (const void*)dq, (const void*)dk, (const void*)dv})
    if (!aligned16(t)) return api_fail(DT_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  dtk::AttnTrainParams a{};
  if ((rc = rate(fn, p, rng, &a.threshold, &a.inv_keep))) return rc;
  int sms = 0;
  if ((rc = need_sm100(fn, &sms, &a.status))) return rc;
  a.q = q, a.k = k, a.v = v, a.o = const_cast<void*>(o), a.lse = const_cast<float*>(lse), a.pad_len = pad_len;
  if (workspace_bytes < attn_workspace(B, S, Hq, Hkv, D, a.threshold != 0, sms) || !aligned16(workspace))
    return api_fail(DT_ERR_INVALID, "%s: workspace of %lld bytes is too small or not 16-byte aligned", fn,
                    (long long)workspace_bytes);
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = static_cast<float*>(workspace);
  a.part = a.delta + delta_elems(B, S, Hq);
  a.grad_max = a.part + attn_part_elems(B, S, Hq, Hkv, D, sms);
  a.grad_parts = dtk::attn_train_grad_parts(S, Hq / Hkv, D);
  const int64_t words = a.threshold ? dtk::attn_train_words(B, S, Hq, D) : 0;
  if (words) a.words = reinterpret_cast<uint32_t*>(a.grad_max), a.grad_max += words;
  long long* const to[24] = {&a.q_sb,  &a.q_ss,  &a.q_sh,  &a.k_sb,  &a.k_ss,  &a.k_sh,  &a.v_sb,  &a.v_ss,
                             &a.v_sh,  &a.o_sb,  &a.o_ss,  &a.o_sh,  &a.do_sb, &a.do_ss, &a.do_sh, &a.dq_sb,
                             &a.dq_ss, &a.dq_sh, &a.dk_sb, &a.dk_ss, &a.dk_sh, &a.dv_sb, &a.dv_ss, &a.dv_sh};
  for (int i = 0; i < 24; ++i) *to[i] = strides[i];
  a.B = B, a.S = S, a.Hq = Hq, a.Hkv = Hkv, a.R = Hq / Hkv;
  a.scale = scale > 0.f ? scale : 1.0f / sqrtf((float)D);
  a.rng = reinterpret_cast<const long long*>(rng);
  a.site = site;
  a.HC = a.R < 64 ? a.R : 64;
  a.PT128 = 128 / a.HC, a.PT64 = 64 / a.HC, a.by_pt64 = dtk::FastDiv((uint32_t)a.PT64);
  const bool bf16 = dtype == DT_DTYPE_BF16;
  dtk::AttnTrainMaps m;
  const uint32_t hc = (uint32_t)a.HC;
  if ((rc = dtk::api_encode_bshd(&m.q_tile, q, bf16, B, S, Hq, D, a.q_sb, a.q_ss, a.q_sh, hc, 128 / hc, "q")) ||
      (rc = dtk::api_encode_groups(&m.q_blk, q, bf16, B, S, Hkv, a.R, D, a.q_sb, a.q_ss, a.q_sh, hc, 64 / hc, "q")) ||
      (rc = dtk::api_encode_bshd(&m.do_tile, dout, bf16, B, S, Hq, D, a.do_sb, a.do_ss, a.do_sh, hc, 128 / hc,
                                 "dout")) ||
      (rc = dtk::api_encode_bshd(&m.o_tile, o, bf16, B, S, Hq, D, a.o_sb, a.o_ss, a.o_sh, hc, 128 / hc, "o")) ||
      (rc = dtk::api_encode_groups(&m.do_blk, dout, bf16, B, S, Hkv, a.R, D, a.do_sb, a.do_ss, a.do_sh, hc, 64 / hc,
                                   "dout")) ||
      (rc = dtk::api_encode_bshd(&m.k_tile, k, bf16, B, S, Hkv, D, a.k_sb, a.k_ss, a.k_sh, 1, 128, "k")) ||
      (rc = dtk::api_encode_bshd(&m.k_blk, k, bf16, B, S, Hkv, D, a.k_sb, a.k_ss, a.k_sh, 1, 64, "k")) ||
      (rc = dtk::api_encode_bshd(&m.v_tile, v, bf16, B, S, Hkv, D, a.v_sb, a.v_ss, a.v_sh, 1, 128, "v")) ||
      (rc = dtk::api_encode_bshd(&m.v_blk, v, bf16, B, S, Hkv, D, a.v_sb, a.v_ss, a.v_sh, 1, 64, "v")))
    return rc;
  return cuda_status(dtk::launch_attn_train_bwd_sm100(a, m, D, bf16, sms, static_cast<cudaStream_t>(stream)), fn);
}

int64_t dt_attn_train_forward_workspace(int B, int S, int Hq, int Hkv, int D) {
  const char* fn = "dt_attn_train_forward_workspace";
  const int64_t s[3] = {8, 8, 8};
  int rc = check_attn(fn, B, S, Hq, Hkv, D, s, 3, DT_DTYPE_BF16);
  int sms = 0;
  if (rc || (rc = need_sm100(fn, &sms))) return -rc;
  return attn_forward_workspace(B, S, Hq, Hkv, D, sms);
}

int64_t dt_attn_train_workspace(int B, int S, int Hq, int Hkv, int D, int has_dropout) {
  const int64_t s[3] = {8, 8, 8};
  int rc = check_attn("dt_attn_train_workspace", B, S, Hq, Hkv, D, s, 3, DT_DTYPE_BF16);
  int sms = 0;
  if (rc || (rc = need_sm100("dt_attn_train_workspace", &sms))) return -rc;
  return attn_workspace(B, S, Hq, Hkv, D, has_dropout != 0, sms);
}

int dt_rope_grad(void* g, int64_t g_stride, int64_t rows, const float* cos_tab, const float* sin_tab,
                 int64_t cos_stride, int cos_rows, int seq_len, int rope_cols, int head_dim, int dtype, void* stream) {
  const char* fn = "dt_rope_grad";
  Range range(fn);
  if (!g || !cos_tab || !sin_tab) return api_fail(DT_ERR_INVALID, "%s: null g/cos/sin pointer", fn);
  if (rows < 1 || seq_len < 1) return api_fail(DT_ERR_INVALID, "%s: sizes must be positive", fn);
  if (head_dim != 32 && head_dim != 64)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: head_dim %d not in {32, 64}", fn, head_dim);
  if (dtype != DT_DTYPE_BF16 && dtype != DT_DTYPE_FP16)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16 or fp16)", fn, dtype);
  if (rope_cols < head_dim || rope_cols % head_dim || g_stride < rope_cols || g_stride % 8 || !aligned16(g))
    return api_fail(DT_ERR_INVALID, "%s: rope_cols %d / row stride %lld / alignment", fn, rope_cols,
                    (long long)g_stride);
  if (cos_rows < seq_len || cos_stride < head_dim || cos_stride % 2 ||
      ((reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) & 7))
    return api_fail(DT_ERR_INVALID, "%s: cos/sin need %d rows of %d, 8-byte aligned", fn, seq_len, head_dim);
  int sms = 0;
  const int rc = need_sm100(fn, &sms);
  if (rc) return rc;
  dtk::RopeGradParams a{};
  a.x = g, a.cos = cos_tab, a.sin = sin_tab, a.stride = g_stride, a.rows = rows, a.cs_stride = cos_stride;
  a.rope_cols = rope_cols, a.head_dim = head_dim, a.seq_len = seq_len;
  return cuda_status(dtk::launch_rope_grad_sm100(a, dtype == DT_DTYPE_BF16, sms, static_cast<cudaStream_t>(stream)),
                     fn);
}

int64_t dt_residual_norm_workspace(int64_t M, int H, int64_t gate_rows, int has_post) {
  if (M < 1 || M > 0x7fffffffLL || H < 1 || H > kMaxHidden || gate_rows < 0 || (gate_rows > 0 && M % gate_rows != 0))
    return -api_fail(DT_ERR_INVALID, "dt_residual_norm_workspace: bad sizes (M=%lld H=%d gate_rows=%lld)", (long long)M,
                     H, (long long)gate_rows);
  int sms = 0;
  const int rc = need_sm100("dt_residual_norm_workspace", &sms);
  if (rc) return -rc;
  // Alignment decides between two plans when the backward call comes: room for either.
  const int64_t a = part_elems(dtk::residual_norm_plan(M, H, gate_rows, true, sms), H, gate_rows, has_post != 0);
  const int64_t b = part_elems(dtk::residual_norm_plan(M, H, gate_rows, false, sms), H, gate_rows, has_post != 0);
  return 4 * (a > b ? a : b);
}

static int check_residual_norm(const char* fn, const void* x, const void* w_pre, const void* gate, int64_t gate_rows,
                               int64_t M, int H, int dtype) {
  int rc = check_dtype(fn, dtype);
  if (rc) return rc;
  if ((rc = check_rows(fn, x, M, H, "M", "H"))) return rc;
  if (H > kMaxHidden) return api_fail(DT_ERR_UNSUPPORTED, "%s: H %d above %d", fn, H, kMaxHidden);
  if (M > 0x7fffffffLL) return api_fail(DT_ERR_UNSUPPORTED, "%s: M %lld above 2^31 - 1", fn, (long long)M);
  if (!w_pre) return api_fail(DT_ERR_INVALID, "%s: null w_pre", fn);
  if (gate && (gate_rows < 1 || M % gate_rows != 0))
    return api_fail(DT_ERR_INVALID, "%s: gate_rows %lld does not divide M %lld", fn, (long long)gate_rows,
                    (long long)M);
  return DT_OK;
}

int dt_residual_norm_forward(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
                             const void* gate, int64_t gate_stride, int64_t gate_rows, const void* w_pre,
                             const void* w_post, void* h, void* n, float* stats, int64_t M, int H, float alpha,
                             float eps, double p, const int64_t* rng, uint32_t site, int dtype, void* stream) {
  const char* fn = "dt_residual_norm_forward";
  Range range(fn);
  int rc = check_residual_norm(fn, x, w_pre, gate, gate_rows, M, H, dtype);
  if (rc) return rc;
  if (!h || !n || !stats) return api_fail(DT_ERR_INVALID, "%s: null h/n/stats", fn);
  if ((rc = check_elem_aligned(fn, dtype, {x, residual, gate, w_pre, w_post, h, n}))) return rc;
  dtk::ResidualNormParams a{};
  if ((rc = rate(fn, p, rng, &a.threshold, &a.inv_keep))) return rc;
  int sms = 0;
  if ((rc = need_sm100(fn, &sms))) return rc;
  a.x = x, a.residual = residual, a.gate = gate, a.w_pre = w_pre, a.w_post = w_post, a.h = h, a.n = n, a.stats = stats;
  a.x_stride = x_stride, a.res_stride = res_stride, a.gate_stride = gate_stride;
  a.M = M, a.H = H, a.gate_rows = gate ? gate_rows : 0, a.by_gate = dtk::FastDiv(gate ? (uint32_t)gate_rows : 1u);
  a.alpha = alpha, a.eps = eps, a.rng = reinterpret_cast<const long long*>(rng), a.site = site;
  return cuda_status(dtk::launch_residual_norm_fwd_sm100(a, dtype, sms, static_cast<cudaStream_t>(stream)), fn);
}

int dt_residual_norm_backward(const void* dh, int64_t dh_stride, const void* dn, int64_t dn_stride, const void* x,
                              int64_t x_stride, const void* residual, int64_t res_stride, const void* gate,
                              int64_t gate_stride, int64_t gate_rows, const void* w_pre, const void* w_post,
                              const float* stats, void* dx, void* dresidual, void* dw_pre, void* dw_post, void* dgate,
                              void* workspace, int64_t workspace_bytes, int64_t M, int H, float alpha, float eps,
                              double p, const int64_t* rng, uint32_t site, int dtype, void* stream) {
  const char* fn = "dt_residual_norm_backward";
  Range range(fn);
  int rc = check_residual_norm(fn, x, w_pre, gate, gate_rows, M, H, dtype);
  if (rc) return rc;
  if (!dh && !dn) return api_fail(DT_ERR_INVALID, "%s: dh and dn are both null", fn);
  if (!stats || !dx || (dn && !dw_pre) || (w_post && !dw_post) || (gate && !dgate))
    return api_fail(DT_ERR_INVALID, "%s: null stats or gradient pointer", fn);
  if ((rc = check_elem_aligned(fn, dtype, {dh, dn, x, residual, gate, w_pre, w_post, dx, dresidual, dw_pre, dw_post,
                                           dgate})))
    return rc;
  dtk::ResidualNormParams a{};
  if ((rc = rate(fn, p, rng, &a.threshold, &a.inv_keep))) return rc;
  int sms = 0;
  if ((rc = need_sm100(fn, &sms))) return rc;
  if (!gate) gate_rows = 0;
  const bool post = w_post != nullptr;
  a.x = x, a.residual = residual, a.gate = gate, a.w_pre = w_pre, a.w_post = w_post, a.dh = dh, a.dn = dn;
  a.stats = const_cast<float*>(stats);
  a.dx = dx, a.dresidual = dresidual, a.dw_pre = dw_pre, a.dw_post = dw_post, a.dgate = dgate;
  a.x_stride = x_stride, a.res_stride = res_stride, a.gate_stride = gate_stride;
  a.dh_stride = dh_stride, a.dn_stride = dn_stride;
  a.M = M, a.H = H, a.gate_rows = gate_rows;
  a.alpha = alpha, a.eps = eps, a.rng = reinterpret_cast<const long long*>(rng), a.site = site;
  const dtk::ResidualNormPlan plan = dtk::residual_norm_plan(M, H, gate_rows, dtk::residual_norm_ring(a, dtype), sms);
  if (workspace_bytes < 4 * part_elems(plan, H, gate_rows, post) || !workspace || !aligned16(workspace))
    return api_fail(DT_ERR_INVALID, "%s: workspace of %lld bytes is too small, null or not 16-byte aligned", fn,
                    (long long)workspace_bytes);
  float* part = static_cast<float*>(workspace);
  const int64_t one = plan.grid > 1 ? plan.grid * (int64_t)H : 0, step = (one + 3) / 4 * 4;
  a.part_pre = part;
  a.part_post = part + step;
  a.part_gate = part + (post ? 2 : 1) * step;
  return cuda_status(dtk::launch_residual_norm_bwd_sm100(a, plan, dtype, static_cast<cudaStream_t>(stream)), fn);
}

int dt_dropout(const void* x, int64_t x_stride, const void* residual, int64_t res_stride, void* y, int64_t y_stride,
               int64_t rows, int cols, double p, const int64_t* rng, uint32_t site, int dtype, void* stream) {
  const char* fn = "dt_dropout";
  Range range(fn);
  int rc = check_dtype(fn, dtype);
  if (rc) return rc;
  if ((rc = check_rows(fn, x, rows, cols, "rows", "cols"))) return rc;
  if (cols > kMaxCols) return api_fail(DT_ERR_UNSUPPORTED, "%s: %d columns, above %d", fn, cols, kMaxCols);
  if (!y) return api_fail(DT_ERR_INVALID, "%s: null y", fn);
  if ((rc = check_elem_aligned(fn, dtype, {x, residual, y}))) return rc;
  dtk::DropoutParams a{};
  if ((rc = rate(fn, p, rng, &a.threshold, &a.inv_keep))) return rc;
  int sms = 0;
  if ((rc = need_sm100(fn, &sms))) return rc;
  a.x = x, a.residual = residual, a.y = y, a.x_stride = x_stride, a.res_stride = res_stride, a.y_stride = y_stride;
  a.rows = rows, a.cols = cols, a.rng = reinterpret_cast<const long long*>(rng), a.site = site;
  return cuda_status(dtk::launch_dropout_sm100(a, dtype, sms, static_cast<cudaStream_t>(stream)), fn);
}

}  // extern "C"
