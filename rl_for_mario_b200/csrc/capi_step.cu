// C-ABI entry points of the end of a training step (include/dt_train.h): the gradient's norm and
// AdamW over many tensors.  Argument validation and dispatch; no entry point allocates device memory.
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>

#include <cfloat>
#include <cmath>

#include "../../include/dt_attn.h"
#include "../../include/dt_train.h"
#include "dt_internal.h"

namespace {

using dtk::api_fail;
using dtk::TensorSlot;

struct Range {
  explicit Range(const char* name) { nvtxRangePushA(name); }
  ~Range() { nvtxRangePop(); }
  Range(const Range&) = delete;
  Range& operator=(const Range&) = delete;
};

constexpr int64_t kMaxBlocks = 0x3fffffffLL;  // of 256 elements, of a launch
constexpr int64_t kMaxSize = 1LL << 37;      // elements of a tensor: fewer blocks than a launch takes

int cuda_status(cudaError_t e, const char* what) {
  return e == cudaSuccess ? DT_OK : api_fail(DT_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

int need_sm100(const char* fn, int* num_sms) {
  int* status = nullptr;
  int cc = 0;
  const int rc = dtk::api_device(&status, &cc, num_sms);
  if (rc) return rc;
  if (cc != 10) return api_fail(DT_ERR_UNSUPPORTED, "%s: needs an sm_100 GPU (current device is cc %d.x)", fn, cc);
  return DT_OK;
}

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// One tensor's arguments; params may be null (the norm).
int check_tensor(const char* fn, int i, int64_t p, int64_t g, int64_t n, int kind, int ngroups) {
  const int dtype = kind & 0xff, group = kind >> 8;
  if (dtype != DT_DTYPE_BF16 && dtype != DT_DTYPE_FP16 && dtype != DT_DTYPE_FP32)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: tensor %d: dtype %d not supported", fn, i, dtype);
  if (kind < 0 || group >= ngroups)
    return api_fail(DT_ERR_INVALID, "%s: tensor %d: group %d of %d", fn, i, group, ngroups);
  if (n < 0 || n >= kMaxSize) return api_fail(DT_ERR_INVALID, "%s: tensor %d: %lld elements", fn, i, (long long)n);
  const int64_t e = dtype == DT_DTYPE_FP32 ? 4 : 2;
  if (p % e || g % e) return api_fail(DT_ERR_INVALID, "%s: tensor %d is not aligned to its elements", fn, i);
  return DT_OK;
}

// Walks through the tensors in launches of up to kMaxTensors tensors and kMaxBlocks blocks: f(slots, count, units, first
// block of all, last launch).  Tensors' units: their elements in units of `unit`, rounded up; blocks: of 256.
template <typename F>
int in_launches(int count, const int64_t* params, const int64_t* grads, const int64_t* sizes, const int32_t* kinds,
                int64_t unit, F f) {
  TensorSlot slots[dtk::kMaxTensors];
  int64_t first = 0;
  for (int i = 0; i < count;) {
    int n = 0;
    int64_t units = 0, blocks = 0;
    for (; i < count && n < dtk::kMaxTensors; ++i, ++n) {
      const int64_t more = (sizes[i] + unit - 1) / unit, b = (sizes[i] + 255) / 256;
      if (blocks + b > kMaxBlocks && n) break;
      units += more;
      slots[n] = TensorSlot{params ? reinterpret_cast<void*>(params[i]) : nullptr, reinterpret_cast<const void*>(grads[i]),
                            sizes[i], (uint32_t)units, (uint32_t)blocks, (uint32_t)kinds[i]};
      blocks += b;
    }
    const int rc = f(slots, n, (uint32_t)units, first, i == count);
    if (rc) return rc;
    first += blocks;
  }
  return DT_OK;
}

// Sums of squares of every launch's blocks behind one another; `parts` of them in all.  norm: of a single block.
int launch_norm(const char* fn, int count, const int64_t* grads, const int64_t* sizes, const int32_t* kinds,
                double* parts, int64_t room, float* norm, int num_sms, cudaStream_t st, int* total) {
  *total = 0;
  return in_launches(count, nullptr, grads, sizes, kinds, dtk::grad_norm_unit(),
                     [&](const TensorSlot* slots, int n, uint32_t units, int64_t, bool) {
                       const int grid = dtk::grad_norm_grid(units, num_sms);
                       if (*total + grid > room) return api_fail(DT_ERR_INVALID, "%s: the workspace is too small", fn);
                       dtk::GradNormParams p{};
                       p.count = n, p.units = units, p.parts = parts + *total;
                       p.norm = n == count && grid == 1 ? norm : nullptr;
                       *total += grid;
                       return cuda_status(dtk::launch_grad_norm_sm100(slots, p, num_sms, st), fn);
                     });
}

int64_t norm_parts(int count, int num_sms) {
  // A launch ends at kMaxTensors tensors, or before one that would pass kMaxBlocks: 2^38 elements, which no GPU holds.
  const int64_t launches = (count + dtk::kMaxTensors - 1) / dtk::kMaxTensors;
  return launches * dtk::grad_norm_grid(kMaxBlocks, num_sms);
}

}  // namespace

extern "C" {

int64_t dt_grad_norm_workspace(int count) {
  const char* fn = "dt_grad_norm_workspace";
  if (count < 1) return -api_fail(DT_ERR_INVALID, "%s: %d tensors", fn, count);
  int sms = 0;
  const int rc = need_sm100(fn, &sms);
  if (rc) return -rc;
  return 8 * norm_parts(count, sms);
}

int dt_grad_norm(int count, const int64_t* tensors, const int64_t* sizes, const int32_t* kinds, float* norm,
                 void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "dt_grad_norm";
  Range range(fn);
  if (count < 1 || !tensors || !sizes || !kinds || !norm || !aligned(norm, 4))
    return api_fail(DT_ERR_INVALID, "%s: %d tensors, or a null pointer", fn, count);
  for (int i = 0; i < count; ++i) {
    const int rc = check_tensor(fn, i, 0, tensors[i], sizes[i], kinds[i], 1);
    if (rc) return rc;
  }
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < 8)
    return api_fail(DT_ERR_INVALID, "%s: workspace null or not 16-byte aligned", fn);
  int sms = 0, parts = 0;
  int rc = need_sm100(fn, &sms);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launch_norm(fn, count, tensors, sizes, kinds, static_cast<double*>(workspace), workspace_bytes / 8, norm, sms, st,
                   &parts);
  if (rc || parts == 1) return rc;
  return cuda_status(dtk::launch_grad_norm_sum_sm100(static_cast<double*>(workspace), parts, norm, st), fn);
}

int dt_adamw_step(int count, const int64_t* params, const int64_t* grads, const int64_t* sizes, const int32_t* kinds,
                  int ngroups, const DtAdamWGroup* groups, int state_bits, void* exp_avg, void* exp_avg_sq,
                  uint8_t* exp_avg_scale, uint8_t* exp_avg_sq_scale, float* master, int64_t* state, uint32_t* ticket,
                  double max_norm, float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "dt_adamw_step";
  Range range(fn);
  if (count < 1 || !params || !grads || !sizes || !kinds || !groups || !exp_avg || !exp_avg_sq || !state || !ticket)
    return api_fail(DT_ERR_INVALID, "%s: %d tensors, or a null pointer", fn, count);
  if (ngroups < 1 || ngroups > dtk::kAdamWGroups)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: %d groups, 1 to %d are taken", fn, ngroups, dtk::kAdamWGroups);
  if (state_bits != 8 && state_bits != 32)
    return api_fail(DT_ERR_UNSUPPORTED, "%s: state_bits %d not in {8, 32}", fn, state_bits);
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale))
    return api_fail(DT_ERR_INVALID, "%s: null scales", fn);
  if (!aligned(exp_avg, 16) || !aligned(exp_avg_sq, 16) || !aligned(master, 16) || !aligned(state, 8) ||
      !aligned(ticket, 4))
    return api_fail(DT_ERR_INVALID, "%s: averages and master must be 16-byte, state 8-byte, ticket 4-byte aligned", fn);
  for (int i = 0; i < ngroups; ++i) {
    const DtAdamWGroup& g = groups[i];
    if (!(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1 && g.lr >= 0 && g.lr < INFINITY &&
          g.weight_decay >= 0 && g.weight_decay < INFINITY && (float)g.eps >= FLT_MIN && (float)g.eps < INFINITY) ||
        !aligned(g.lr_tensor, 4))
      return api_fail(DT_ERR_INVALID, "%s: group %d: lr %g, betas %g %g, eps %g, weight_decay %g", fn, i, g.lr, g.beta1,
                      g.beta2, g.eps, g.weight_decay);
  }
  for (int i = 0; i < count; ++i) {
    const int rc = check_tensor(fn, i, params[i], grads[i], sizes[i], kinds[i], ngroups);
    if (rc) return rc;
    if (sizes[i] && !params[i]) return api_fail(DT_ERR_INVALID, "%s: tensor %d is null", fn, i);
  }
  const bool clip = max_norm > 0;
  if (std::isnan(max_norm) || (clip && (!((float)max_norm > 0.f) || !norm || !aligned(norm, 4) || !workspace ||
                                        !aligned(workspace, 16))))
    return api_fail(DT_ERR_INVALID, "%s: max_norm %g needs norm and a 16-byte aligned workspace", fn, max_norm);
  dtk::AdamWParams p{};
  int rc = need_sm100(fn, &p.nparts);
  if (rc) return rc;
  const int sms = p.nparts;
  p.nparts = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (clip) {
    rc = launch_norm(fn, count, grads, sizes, kinds, static_cast<double*>(workspace), workspace_bytes / 8, nullptr, sms,
                     st, &p.nparts);
    if (rc) return rc;
    p.parts = static_cast<const double*>(workspace), p.norm = norm, p.max_norm = (float)max_norm;
  }
  for (int i = 0; i < ngroups; ++i) {
    const DtAdamWGroup& g = groups[i];
    p.group[i] = dtk::AdamWGroup{g.lr, g.beta1, g.beta2, g.eps, g.weight_decay, g.lr_tensor};
  }
  p.one = 1.f;
  p.ngroups = ngroups, p.m = exp_avg, p.v = exp_avg_sq, p.master = master;
  if (state_bits == 8) p.m_scale = exp_avg_scale, p.v_scale = exp_avg_sq_scale;
  p.state = reinterpret_cast<long long*>(state);
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) blocks += (sizes[i] + 255) / 256;
  p.pairs = dtk::adamw_pairs(blocks, state_bits, sms);
  return in_launches(count, params, grads, sizes, kinds, 512LL * p.pairs,
                     [&](const TensorSlot* slots, int n, uint32_t units, int64_t first, bool last) {
                       p.count = n, p.units = units, p.first = first, p.ticket = last ? ticket : nullptr;
                       return cuda_status(dtk::launch_adamw_sm100(slots, p, sms, st), fn);
                     });
}

int dt_adamw_moments(const uint8_t* exp_avg, const uint8_t* exp_avg_scale, const uint8_t* exp_avg_sq,
                     const uint8_t* exp_avg_sq_scale, int64_t blocks, void* exp_avg_out, void* exp_avg_sq_out,
                     void* stream) {
  const char* fn = "dt_adamw_moments";
  Range range(fn);
  if (!exp_avg || !exp_avg_scale || !exp_avg_sq || !exp_avg_sq_scale || !exp_avg_out || !exp_avg_sq_out || blocks < 1)
    return api_fail(DT_ERR_INVALID, "%s: %lld blocks, or a null pointer", fn, (long long)blocks);
  if (!aligned(exp_avg, 16) || !aligned(exp_avg_sq, 16) || !aligned(exp_avg_out, 16) || !aligned(exp_avg_sq_out, 16))
    return api_fail(DT_ERR_INVALID, "%s: codes and outputs must be 16-byte aligned", fn);
  int sms = 0;
  const int rc = need_sm100(fn, &sms);
  if (rc) return rc;
  return cuda_status(dtk::launch_adamw_moments_sm100(exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale, blocks,
                                                     exp_avg_out, exp_avg_sq_out, sms, static_cast<cudaStream_t>(stream)),
                     fn);
}

}  // extern "C"
