// Dropout with a mask that is never stored (philox.cuh), optionally added to a
// residual:  y = residual + x * m / (1 - p).  The backward pass is the same
// kernel on the gradient, without a residual.
//
// Bound by HBM: 2 (or 3 with a residual) elements of traffic each, against some
// fourteen integer instructions for each element of mask and its use, which have to
// fit under the loads: 16-bit pairs are dropped by one AND with a mask of the word
// that decides on them (73,728 x 2,048 bf16, 604 MB: 91 us = 6.6 TB/s; with a bit,
// a test and a select for each element 111 us).  A warp takes 256 columns of one
// row; rows that are contiguous, 16-byte aligned and a multiple of 8 wide are walked
// as one long row.
#include "dt_common.cuh"
#include "dt_internal.h"
#include "train_common.cuh"

namespace dtk {

namespace {

constexpr int kTurn = 2;  // vectors a thread has in flight (73,728 x 2,048 bf16: 92.3 us with one, 91.2, 94.1 with four)

// LINEAR: rows follow one another without gaps and their width is a multiple of
// 8, so counter blocks and 8-element vectors are both numbered straight through.
template <int DT, bool LINEAR>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutParams p) {
  using T = typename TrainElem<DT>::T;
  const int lane = threadIdx.x & 31;
  DropKey key{};
  if (p.threshold) key = drop_key(p.rng, p.site);  // p = 0 keeps every word, whatever the key
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  const long long nwarps = (long long)gridDim.x * (blockDim.x >> 5);
  const long long warp0 = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if constexpr (LINEAR) {
    const long long nblk = p.rows * (long long)(p.cols >> 3);
    const long long step = nwarps * 32;
    for (long long i = warp0 * 32 + lane; i < nblk; i += kTurn * step) {
      // kTurn vectors a turn: their loads are in flight together, behind the generator.
      Raw8<DT, true> a[kTurn], r[kTurn];
#pragma unroll
      for (int j = 0; j < kTurn; ++j) {
        if (i + j * step >= nblk) continue;
        a[j].load(x + (i + j * step) * 8, 0, 0, 8);
        if (res) r[j].load(res + (i + j * step) * 8, 0, 0, 8);
      }
#pragma unroll
      for (int j = 0; j < kTurn; ++j) {
        const long long at = i + j * step;
        if (at >= nblk) continue;
        F8 v, add;
        if constexpr (DT == 2) {
          const uint32_t m = keep_bits(key, (unsigned long long)at, p.threshold);
          a[j].get(v.as());
          v.keep(m);
        } else {
          const uint4 m = keep_masks(key, (unsigned long long)at, p.threshold);
          a[j].u.x &= m.x, a[j].u.y &= m.y, a[j].u.z &= m.z, a[j].u.w &= m.w;
          a[j].get(v.as());
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v.p[e] = fmul2(v.p[e], both(p.inv_keep));
        if (res) {
          r[j].get(add.as());
#pragma unroll
          for (int e = 0; e < 4; ++e) v.p[e] = fadd2(v.p[e], add.p[e]);
        }
        store8<DT, true>(y + at * 8, 0, 0, 8, v.as());
      }
    }
  } else {
    const int chunks = (p.cols + 255) >> 8;  // 256-column pieces of a row
    const long long total = p.rows * chunks;
    const long long per_row = (p.cols + 7) >> 3;
    for (long long i = warp0; i < total; i += nwarps) {
      const long long row = i / chunks;
      const int w = (int)(i - row * chunks);
      float a[8], r[8];
      load8<DT, false>(x + row * p.x_stride, w, lane, p.cols, a);
      if (res) load8<DT, false>(res + row * p.res_stride, w, lane, p.cols, r);
      const uint32_t m = keep8<false>(key, (unsigned long long)(row * per_row), w, lane, p.threshold);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = (m >> e) & 1u ? a[e] * p.inv_keep : 0.f;
      if (res)
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += r[e];
      store8<DT, false>(y + row * p.y_stride, w, lane, p.cols, a);
    }
  }
}

template <int DT>
cudaError_t launch(const DropoutParams& p, int num_sms, cudaStream_t st) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y) |
                         reinterpret_cast<uintptr_t>(p.residual);
  const bool linear = p.cols % 8 == 0 && (bits & 15) == 0 && (p.rows == 1 || (p.x_stride == p.cols &&
                      p.y_stride == p.cols && (!p.residual || p.res_stride == p.cols)));
  const long long warps = linear ? (p.rows * (p.cols >> 3) + 32 * kTurn - 1) / (32 * kTurn) : p.rows * ((p.cols + 255) >> 8);
  const long long want = (warps + 7) / 8, cap = (long long)num_sms * 64;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (linear)
    dropout_kernel<DT, true><<<grid, 256, 0, st>>>(p);
  else
    dropout_kernel<DT, false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_dropout_sm100(const DropoutParams& p, int dtype, int num_sms, cudaStream_t st) {
  if (dtype == 0) return launch<0>(p, num_sms, st);
  if (dtype == 1) return launch<1>(p, num_sms, st);
  return launch<2>(p, num_sms, st);
}

}  // namespace dtk
