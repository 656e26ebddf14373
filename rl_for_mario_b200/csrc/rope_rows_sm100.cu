// Gradient of the rotate-half RoPE of a projection's q and k heads, in place:
// the forward pass (dt_qkv_rope's epilogue) forms
//   y0 = x0 cos[d] - x1 sin[d],  y1 = x1 cos[d'] + x0 sin[d'],  d' = d + D / 2,
// so  dx0 = dy0 cos[d] + dy1 sin[d'],  dx1 = dy1 cos[d'] - dy0 sin[d].
// One thread takes eight d of one head of one row, 16-byte accesses; bound by
// HBM (2 bytes read and written per element; 96 x 768 rows, 16 heads of 64, 302 MB:
// 53 us = 5.7 TB/s; the tables stay in L1 and L2).  fp32 arithmetic, one rounding.
#include "dt_common.cuh"
#include "dt_internal.h"

namespace dtk {

namespace {

template <bool BF16>
__global__ void __launch_bounds__(256) rope_grad_kernel(const RopeGradParams p) {
  using E = Elem<BF16>;
  const int half = p.head_dim >> 4;           // 16-byte chunks in half a head
  const int per_row = (p.rope_cols >> 4);     // chunk pairs in a row
  const long long total = p.rows * per_row;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long row = i / per_row;
    const int c = (int)(i - row * per_row), head = c / half, d = (c - head * half) * 8;
    const int s = (int)(row % p.seq_len);
    uint4* a = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.x) + row * p.stride + head * p.head_dim + d);
    uint4* b = a + half;
    const float* cr = p.cos + (long long)s * p.cs_stride + d;
    const float* sr = p.sin + (long long)s * p.cs_stride + d;
    const uint4 ua = *a, ub = *b;
    const uint32_t xa[4] = {ua.x, ua.y, ua.z, ua.w}, xb[4] = {ub.x, ub.y, ub.z, ub.w};
    uint32_t ya[4], yb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = E::to_f2(xa[e]), g = E::to_f2(xb[e]);
      const float2 c0 = __ldg(reinterpret_cast<const float2*>(cr) + e);
      const float2 s0 = __ldg(reinterpret_cast<const float2*>(sr) + e);
      const float2 c1 = __ldg(reinterpret_cast<const float2*>(cr + (p.head_dim >> 1)) + e);
      const float2 s1 = __ldg(reinterpret_cast<const float2*>(sr + (p.head_dim >> 1)) + e);
      ya[e] = E::from_f2(f.x * c0.x + g.x * s1.x, f.y * c0.y + g.y * s1.y);
      yb[e] = E::from_f2(g.x * c1.x - f.x * s0.x, g.y * c1.y - f.y * s0.y);
    }
    *a = make_uint4(ya[0], ya[1], ya[2], ya[3]);
    *b = make_uint4(yb[0], yb[1], yb[2], yb[3]);
  }
}

}  // namespace

cudaError_t launch_rope_grad_sm100(const RopeGradParams& p, bool bf16, int num_sms, cudaStream_t st) {
  const long long want = (p.rows * (p.rope_cols >> 4) + 255) / 256, cap = (long long)num_sms * 32;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (bf16)
    rope_grad_kernel<true><<<grid, 256, 0, st>>>(p);
  else
    rope_grad_kernel<false><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dtk
