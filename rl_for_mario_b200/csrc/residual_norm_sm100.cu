// Residual add with the norms before and after it, a gate and dropout, and its
// gradient: what stands between two blocks' products in training, one pass.
//
//   u = x * r_post * w_post   r_post = rsqrt(mean(x^2) + eps)   (u = x without a post norm)
//   v = m u / (1 - p)         m the dropout mask (philox.cuh)
//   h = residual + alpha * g * v
//   n = h * r_pre * w_pre     r_pre = rsqrt(mean(h^2) + eps)
//
// Backward, from dh (the gradient that reaches h past this op) and dn:
//   t  = dn * w_pre,  c = mean(t * h r_pre)
//   D  = dh + r_pre (t - h r_pre c)          the gradient of h: d(residual) = D
//   dg = alpha v D (summed over the rows that share a gate),  dv = alpha g D,  du = m dv / (1 - p)
//   s  = du * w_post, d(x) = r_post (s - x r_post mean(s * x r_post))     (d(x) = du without a post norm)
//   dw_pre = sum over rows of dn h r_pre,  dw_post = sum over rows of du x r_post
// h is formed again from x and residual in fp32 instead of being read back: the
// same bytes, and the gradient does not see the rounding of the stored h.
//
// Everything between the loads and the stores is fp32; each output is rounded
// once, and n is the norm of the unrounded h.
//
// Bound by HBM.  A row is held by WPR = ceil(H / 256) warps, eight columns a
// thread, so it is read once and its sums are a shuffle tree plus (WPR > 1)
// one named barrier; a 256-thread block holds 8 / WPR rows.  The sums over rows
// stay in registers (a thread owns its columns for every row that it meets),
// each block writes one partial row of them and a second kernel adds the
// partial rows in a fixed order: no atomics, the same bits every run.
#include "dt_common.cuh"
#include "dt_internal.h"
#include "train_common.cuh"

namespace dtk {

namespace {

// Sum over the row's warps.  Slots alternate between two halves of `red`, so
// one barrier is enough: a slot is written again two sums later, and the sum
// between has passed a barrier after every read of it.
__device__ __forceinline__ float row_sum(float v, float* red, int& turn, int wpr, int w, int lane, int bar) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (wpr == 1) return v;
  float* slot = red + turn * 32;
  turn ^= 1;
  if (lane == 0) slot[w] = v;
  named_bar_sync(bar, wpr * 32);
  v = 0.f;
  for (int i = 0; i < wpr; ++i) v += slot[i];
  return v;
}

struct RowPlace {
  int w, lane, group, groups, bar;
  float* red;
};

__device__ __forceinline__ RowPlace place(int wpr, float* red_all) {
  RowPlace r;
  const int warp = threadIdx.x >> 5;
  r.group = warp / wpr;
  r.groups = (int)(blockDim.x >> 5) / wpr;
  r.w = warp - r.group * wpr;
  r.lane = threadIdx.x & 31;
  r.bar = 1 + r.group;
  r.red = red_all + r.group * 64;
  return r;
}

// MAXT: the block's largest size, 256 for rows of up to 2048 columns (so that the
// compiler may use more registers), else 1024.
template <int DT, bool VEC, bool POST, bool DROP, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_norm_fwd_kernel(const ResidualNormParams p) {
  using T = typename TrainElem<DT>::T;
  __shared__ float red_all[8 * 64];
  const RowPlace at = place(p.wpr, red_all);
  int turn = 0;
  const int w = at.w, lane = at.lane, H = p.H;
  DropKey key{};
  if constexpr (DROP) key = drop_key(p.rng, p.site);
  const unsigned per_row = (unsigned)(H + 7) >> 3;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* gate = static_cast<const T*>(p.gate);
  float wpre[8], wpost[8];
  load8<DT, VEC>(static_cast<const T*>(p.w_pre), w, lane, H, wpre);
  if constexpr (POST) load8<DT, VEC>(static_cast<const T*>(p.w_post), w, lane, H, wpost);
  const float inv_h = 1.f / (float)H;
  for (long long row = (long long)blockIdx.x * at.groups + at.group; row < p.M; row += (long long)gridDim.x * at.groups) {
    float v[8], h[8], g[8];
    load8<DT, VEC>(x + row * p.x_stride, w, lane, H, v);
    if (res)
      load8<DT, VEC>(res + row * p.res_stride, w, lane, H, h);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = 0.f;
    if (gate) {
      load8<DT, VEC>(gate + (row / p.gate_rows) * p.gate_stride, w, lane, H, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] *= p.alpha;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = p.alpha;
    }
    if constexpr (POST) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
      ss = row_sum(ss, at.red, turn, p.wpr, w, lane, at.bar);
      const float r = rsqrtf(fmaf(ss, inv_h, p.eps));
      if (w == 0 && lane == 0) p.stats[2 * row] = r;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= r * wpost[i];
    }
    if constexpr (DROP) {
      const uint32_t m = keep8<VEC>(key, (unsigned long long)row * per_row, w, lane, p.threshold);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (m >> i) & 1u ? v[i] * p.inv_keep : 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] = fmaf(g[i], v[i], h[i]);
      ss = fmaf(h[i], h[i], ss);
    }
    store8<DT, VEC>(static_cast<T*>(p.h) + row * H, w, lane, H, h);
    ss = row_sum(ss, at.red, turn, p.wpr, w, lane, at.bar);
    const float r = rsqrtf(fmaf(ss, inv_h, p.eps));
    if (w == 0 && lane == 0) p.stats[2 * row + 1] = r;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= r * wpre[i];
    store8<DT, VEC>(static_cast<T*>(p.n) + row * H, w, lane, H, h);
  }
}

// Adds the groups' accumulators (fixed order) and writes the block's row of
// them: fp32 into `part`, or the finished gradient into `out`.
template <int DT, bool VEC>
__device__ __forceinline__ void flush_row(float (&acc)[8], float* sh, const RowPlace& at, int H, float* part,
                                          typename TrainElem<DT>::T* out) {
  __syncthreads();  // earlier readers of `sh` are done
  const int width = at.groups > 1 ? (int)(blockDim.x / at.groups) * 8 : 0;
  if (at.groups > 1) {
    if (at.group > 0) {
      float* mine = sh + (at.group - 1) * width + at.w * 256;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i * 32 + at.lane] = acc[i];
    }
    __syncthreads();
    if (at.group == 0)
      for (int q = 1; q < at.groups; ++q) {
        const float* theirs = sh + (q - 1) * width + at.w * 256;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += theirs[i * 32 + at.lane];
      }
  }
  if (at.group == 0) {
    if (part)
      store8<2, VEC>(part, at.w, at.lane, H, acc);
    else
      store8<DT, VEC>(out, at.w, at.lane, H, acc);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
}

// Rows are cut into spans (the rows that share a row of the gate; all rows when
// there is no gate or each row has its own) and these into chunks; a block walks
// chunks blockIdx.x, blockIdx.x + gridDim.x, ... and flushes the gate's sum at
// the end of each, the weights' sums at its own end.
template <int DT, bool VEC, bool POST, bool DROP, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_norm_bwd_kernel(const ResidualNormParams p) {
  using T = typename TrainElem<DT>::T;
  __shared__ float red_all[8 * 64];
  __shared__ float sums[7 * 256];
  const RowPlace at = place(p.wpr, red_all);
  int turn = 0;
  const int w = at.w, lane = at.lane, H = p.H;
  DropKey key{};
  if constexpr (DROP) key = drop_key(p.rng, p.site);
  const unsigned per_row = (unsigned)(H + 7) >> 3;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* gate = static_cast<const T*>(p.gate);
  const T* dh = static_cast<const T*>(p.dh);
  const T* dn = static_cast<const T*>(p.dn);
  T* dgate = static_cast<T*>(p.dgate);
  float wpre[8], wpost[8], a_pre[8], a_post[8], a_gate[8];
  load8<DT, VEC>(static_cast<const T*>(p.w_pre), w, lane, H, wpre);
  if constexpr (POST) load8<DT, VEC>(static_cast<const T*>(p.w_post), w, lane, H, wpost);
#pragma unroll
  for (int i = 0; i < 8; ++i) a_pre[i] = a_post[i] = a_gate[i] = 0.f;
  const float inv_h = 1.f / (float)H;
  const bool sum_gate = gate && p.gate_rows > 1;

  for (long long chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    const long long span = chunk / p.chunks_per_span;  // the gate's row, when several rows share it
    const long long r0 = span * p.span_rows + (chunk - span * p.chunks_per_span) * p.chunk_rows;
    const long long r1 = min(r0 + p.chunk_rows, (span + 1) * p.span_rows);
    for (long long row = r0 + at.group; row < r1; row += at.groups) {
      float xv[8], h[8], g[8], d[8], t[8];
      load8<DT, VEC>(x + row * p.x_stride, w, lane, H, xv);
      if (res)
        load8<DT, VEC>(res + row * p.res_stride, w, lane, H, h);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = 0.f;
      if (dh)
        load8<DT, VEC>(dh + row * p.dh_stride, w, lane, H, d);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
      if (dn) load8<DT, VEC>(dn + row * p.dn_stride, w, lane, H, t);
      if (gate) {
        load8<DT, VEC>(gate + (sum_gate ? span : row) * p.gate_stride, w, lane, H, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= p.alpha;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = p.alpha;
      }
      float v[8];
      float r_post = 1.f;
      if constexpr (POST) {
        r_post = p.stats[2 * row];
#pragma unroll
        for (int i = 0; i < 8; ++i) xv[i] *= r_post;  // from here on the normalised x
      }
      uint32_t m = 0xffu;
      if constexpr (DROP) m = keep8<VEC>(key, (unsigned long long)row * per_row, w, lane, p.threshold);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float u = xv[i];
        if constexpr (POST) u *= wpost[i];
        if constexpr (DROP) u = (m >> i) & 1u ? u * p.inv_keep : 0.f;
        v[i] = u;
      }
      if (dn) {
        const float r_pre = p.stats[2 * row + 1];
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[i] = fmaf(g[i], v[i], h[i]) * r_pre;  // the normalised h
          a_pre[i] = fmaf(t[i], h[i], a_pre[i]);
          t[i] *= wpre[i];
          c = fmaf(t[i], h[i], c);
        }
        c = row_sum(c, at.red, turn, p.wpr, w, lane, at.bar) * inv_h;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fmaf(r_pre, fmaf(-h[i], c, t[i]), d[i]);
      }
      if (p.dresidual) store8<DT, VEC>(static_cast<T*>(p.dresidual) + row * H, w, lane, H, d);
      if (gate) {
        if (sum_gate) {
#pragma unroll
          for (int i = 0; i < 8; ++i) a_gate[i] = fmaf(p.alpha * v[i], d[i], a_gate[i]);
        } else {
          float dg[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) dg[i] = p.alpha * v[i] * d[i];
          store8<DT, VEC>(dgate + row * H, w, lane, H, dg);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d[i] *= g[i];
        if constexpr (DROP) d[i] = (m >> i) & 1u ? d[i] * p.inv_keep : 0.f;
      }
      if constexpr (POST) {
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a_post[i] = fmaf(d[i], xv[i], a_post[i]);
          d[i] *= wpost[i];
          c = fmaf(d[i], xv[i], c);
        }
        c = row_sum(c, at.red, turn, p.wpr, w, lane, at.bar) * inv_h;
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = r_post * fmaf(-xv[i], c, d[i]);
      }
      store8<DT, VEC>(static_cast<T*>(p.dx) + row * H, w, lane, H, d);
    }
    if (sum_gate) {
      const bool whole = p.chunks_per_span == 1;
      flush_row<DT, VEC>(a_gate, sums, at, H, whole ? nullptr : p.part_gate + chunk * H, whole ? dgate + span * H : nullptr);
    }
  }
  const bool alone = gridDim.x == 1;
  if (dn)
    flush_row<DT, VEC>(a_pre, sums, at, H, alone ? nullptr : p.part_pre + (long long)blockIdx.x * H,
                       static_cast<T*>(p.dw_pre));
  if constexpr (POST)
    flush_row<DT, VEC>(a_post, sums, at, H, alone ? nullptr : p.part_post + (long long)blockIdx.x * H,
                       static_cast<T*>(p.dw_post));
}

// Adds partial rows: out[j][c] = sum over i < n of part[(j * n + i) * H + c].
// 32 columns and 16 slices of the rows a block, added in a fixed order.
struct SumJob {
  const float* part;
  void* out;
  long long n, rows;  // partial rows of each output row; output rows
};
template <int DT>
__global__ void __launch_bounds__(512) sum_rows_kernel(SumJob a, SumJob b, SumJob c, int H) {
  using T = typename TrainElem<DT>::T;
  __shared__ float sh[16][33];
  const SumJob job = blockIdx.z == 0 ? a : blockIdx.z == 1 ? b : c;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  for (long long j = blockIdx.y; j < job.rows; j += gridDim.y) {
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (col < H) {
      const float* q = job.part + j * job.n * H + col;
      long long i = slice;
      for (; i + 48 < job.n; i += 64) {
        s0 += q[i * H];
        s1 += q[(i + 16) * H];
        s2 += q[(i + 32) * H];
        s3 += q[(i + 48) * H];
      }
      for (; i < job.n; i += 16) s0 += q[i * H];
    }
    sh[slice][lane] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (slice == 0 && col < H) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += sh[i][lane];
      static_cast<T*>(job.out)[j * H + col] = TrainElem<DT>::from_f(s);
    }
    __syncthreads();
  }
}

template <int DT, bool VEC, bool POST>
cudaError_t launch_fwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  if (block > 256) {
    if (p.threshold)
      residual_norm_fwd_kernel<DT, VEC, POST, true, 1024><<<grid, block, 0, st>>>(p);
    else
      residual_norm_fwd_kernel<DT, VEC, POST, false, 1024><<<grid, block, 0, st>>>(p);
  } else {
    if (p.threshold)
      residual_norm_fwd_kernel<DT, VEC, POST, true, 256><<<grid, block, 0, st>>>(p);
    else
      residual_norm_fwd_kernel<DT, VEC, POST, false, 256><<<grid, block, 0, st>>>(p);
  }
  return cudaGetLastError();
}
template <int DT, bool VEC, bool POST>
cudaError_t launch_bwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  if (block > 256) {
    if (p.threshold)
      residual_norm_bwd_kernel<DT, VEC, POST, true, 1024><<<grid, block, 0, st>>>(p);
    else
      residual_norm_bwd_kernel<DT, VEC, POST, false, 1024><<<grid, block, 0, st>>>(p);
  } else {
    if (p.threshold)
      residual_norm_bwd_kernel<DT, VEC, POST, true, 256><<<grid, block, 0, st>>>(p);
    else
      residual_norm_bwd_kernel<DT, VEC, POST, false, 256><<<grid, block, 0, st>>>(p);
  }
  return cudaGetLastError();
}

// 16-byte accesses need every row on a 16-byte boundary and whole vectors.
bool can_vector(const ResidualNormParams& p, int dtype, bool bwd) {
  const long long e = dtype == 2 ? 4 : 2;
  if (p.H % 8) return false;
  const void* ptrs[] = {p.x, p.residual, p.gate, p.w_pre, p.w_post, bwd ? p.dh : p.h, bwd ? p.dn : p.n, p.dx,
                        p.dresidual, p.dgate, p.dw_pre, p.dw_post};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return false;
  const long long strides[] = {p.x_stride, p.residual ? p.res_stride : 0, p.gate ? p.gate_stride : 0,
                               p.dh ? p.dh_stride : 0, p.dn ? p.dn_stride : 0};
  for (long long s : strides)
    if (s * e % 16) return false;
  return true;
}

}  // namespace

// Warps that hold a row (eight columns a thread), rows that a block holds.
static int rn_wpr(int H) { return (H + 255) / 256; }
static int rn_groups(int H) { return rn_wpr(H) >= 8 ? 1 : 8 / rn_wpr(H); }

// Chunks of the backward pass: about six blocks' worth of work for each SM, never
// across two spans.  gate_rows: rows that share a row of the gate, 0 without one.
ResidualNormPlan residual_norm_plan(long long M, int H, long long gate_rows, int num_sms) {
  ResidualNormPlan q;
  const int groups = rn_groups(H);
  q.span_rows = gate_rows > 1 ? gate_rows : M;
  const long long spans = M / q.span_rows;
  const long long want = (long long)num_sms * (rn_wpr(H) > 8 ? 2 : 6);
  const long long most = (q.span_rows + groups - 1) / groups;
  long long per_span = (want + spans - 1) / spans;
  if (per_span > most) per_span = most;
  q.chunk_rows = (q.span_rows + per_span - 1) / per_span;
  q.chunks_per_span = (q.span_rows + q.chunk_rows - 1) / q.chunk_rows;
  q.chunks = spans * q.chunks_per_span;
  q.grid = q.chunks < want ? q.chunks : want;
  return q;
}

cudaError_t launch_residual_norm_fwd_sm100(ResidualNormParams p, int dtype, int num_sms, cudaStream_t st) {
  p.wpr = rn_wpr(p.H);
  const int groups = rn_groups(p.H);
  const unsigned block = (unsigned)(p.wpr * groups * 32);
  const long long want = (p.M + groups - 1) / groups, cap = (long long)num_sms * 32;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  const bool vec = can_vector(p, dtype, false), post = p.w_post != nullptr;
#define DT_FWD(DT)                                                                             \
  return vec ? (post ? launch_fwd<DT, true, true>(p, grid, block, st) : launch_fwd<DT, true, false>(p, grid, block, st)) \
             : (post ? launch_fwd<DT, false, true>(p, grid, block, st) : launch_fwd<DT, false, false>(p, grid, block, st))
  if (dtype == 0) DT_FWD(0);
  if (dtype == 1) DT_FWD(1);
  DT_FWD(2);
#undef DT_FWD
}

cudaError_t launch_residual_norm_bwd_sm100(ResidualNormParams p, const ResidualNormPlan& plan, int dtype,
                                           cudaStream_t st) {
  p.wpr = rn_wpr(p.H);
  const unsigned block = (unsigned)(p.wpr * rn_groups(p.H) * 32), grid = (unsigned)plan.grid;
  p.chunks = plan.chunks;
  p.chunk_rows = plan.chunk_rows;
  p.chunks_per_span = plan.chunks_per_span;
  p.span_rows = plan.span_rows;
  const bool sum_gate = p.gate && p.gate_rows > 1;
  const bool vec = can_vector(p, dtype, true), post = p.w_post != nullptr;
  cudaError_t e;
#define DT_BWD(DT)                                                                             \
  e = vec ? (post ? launch_bwd<DT, true, true>(p, grid, block, st) : launch_bwd<DT, true, false>(p, grid, block, st)) \
          : (post ? launch_bwd<DT, false, true>(p, grid, block, st) : launch_bwd<DT, false, false>(p, grid, block, st))
  if (dtype == 0) DT_BWD(0);
  else if (dtype == 1) DT_BWD(1);
  else DT_BWD(2);
#undef DT_BWD
  if (e != cudaSuccess) return e;
  // What the blocks left in parts.
  SumJob jobs[3];
  int n = 0;
  if (grid > 1 && p.dn) jobs[n++] = SumJob{p.part_pre, p.dw_pre, (long long)grid, 1};
  if (grid > 1 && post) jobs[n++] = SumJob{p.part_post, p.dw_post, (long long)grid, 1};
  if (sum_gate && plan.chunks_per_span > 1)
    jobs[n++] = SumJob{p.part_gate, p.dgate, plan.chunks_per_span, plan.chunks / plan.chunks_per_span};
  if (!n) return cudaSuccess;
  long long rows = 1;
  for (int i = 0; i < n; ++i) rows = jobs[i].rows > rows ? jobs[i].rows : rows;
  for (int i = n; i < 3; ++i) jobs[i] = jobs[0];
  const dim3 g((unsigned)((p.H + 31) / 32), (unsigned)(rows < 4096 ? rows : 4096), (unsigned)n);
  if (dtype == 0) sum_rows_kernel<0><<<g, 512, 0, st>>>(jobs[0], jobs[1], jobs[2], p.H);
  else if (dtype == 1) sum_rows_kernel<1><<<g, 512, 0, st>>>(jobs[0], jobs[1], jobs[2], p.H);
  else sum_rows_kernel<2><<<g, 512, 0, st>>>(jobs[0], jobs[1], jobs[2], p.H);
  return cudaGetLastError();
}

}  // namespace dtk
