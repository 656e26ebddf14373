// The norm of every query and key head with the rotate-half position rotation in
// the same pass, and its gradient.  A head x of D numbers (D even, h = D / 2) at
// position t:
//
//   r = rsqrt(mean(x^2) + eps),  y = x r w          (one w for query heads, one for key heads)
//   o[i]     = y[i] cos[t, i]         - y[i + h] sin[t, i]
//   o[i + h] = y[i + h] cos[t, i + h] + y[i] sin[t, i + h]      i < h
//
// Backward, from g = d(o), with x^ = x r:
//   dy[i] = g[i] cos[t, i] + g[i + h] sin[t, i + h],  dy[i + h] = g[i + h] cos[t, i + h] - g[i] sin[t, i]
//   u = dy w,  dx = r (u - x^ mean(u x^)),  dw = sum over heads and positions of dy x^
// r is taken again from x, which the backward pass reads anyway; nothing is kept between
// the two passes.
//
// Bound by HBM: forward reads and writes each element once, backward reads two and writes
// one.  A head is held by a group of G lanes (a power of two), four pairs (i, i + h) a lane,
// so that the rotation needs no exchange; the row sums are log2 G shuffles.  A group walks
// through some heads of one position with the position's table row and the weights in
// registers, the next head's loads in flight.
#include <type_traits>

#include "dt_common.cuh"
#include "dt_internal.h"
#include "train_common.cuh"

namespace dtk {

namespace {

constexpr int kThreads = 256;

// Four pairs of a head as fp32: a[j], b[j] are elements i, i + h of the lane's pair j.
// VEC: pairs 4 c .. 4 c + 3 of lane c (D a multiple of 8, 4 elements an access); otherwise
// pairs c + G j, those at or past h reading as 0 and not written.
struct Pairs {
  float a[4], b[4];
};

// A head's elements as they stand in memory, on their way while another head is worked on.
template <int DT, bool VEC>
struct RawPairs {
  using T = typename TrainElem<DT>::T;
  T a[4], b[4];
  __device__ __forceinline__ void load(const T* x, int c, int lg, int h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = c + (j << lg);
      a[j] = i < h ? x[i] : TrainElem<DT>::from_f(0.f);
      b[j] = i < h ? x[i + h] : TrainElem<DT>::from_f(0.f);
    }
  }
  __device__ __forceinline__ Pairs get() const {
    Pairs p;
#pragma unroll
    for (int j = 0; j < 4; ++j) p.a[j] = TrainElem<DT>::to_f(a[j]), p.b[j] = TrainElem<DT>::to_f(b[j]);
    return p;
  }
};
template <int DT>
struct RawPairs<DT, true> {
  using T = typename TrainElem<DT>::T;
  using V = typename std::conditional<DT == 2, float4, uint2>::type;
  V a, b;
  __device__ __forceinline__ void load(const T* x, int c, int, int h) {
    a = *reinterpret_cast<const V*>(x + 4 * c);
    b = *reinterpret_cast<const V*>(x + 4 * c + h);
  }
  __device__ __forceinline__ Pairs get() const {
    Pairs p;
    if constexpr (DT == 2) {
      p.a[0] = a.x, p.a[1] = a.y, p.a[2] = a.z, p.a[3] = a.w;
      p.b[0] = b.x, p.b[1] = b.y, p.b[2] = b.z, p.b[3] = b.w;
    } else {
      using E = Elem<DT == 0>;
      const float2 a0 = E::to_f2(a.x), a1 = E::to_f2(a.y), b0 = E::to_f2(b.x), b1 = E::to_f2(b.y);
      p.a[0] = a0.x, p.a[1] = a0.y, p.a[2] = a1.x, p.a[3] = a1.y;
      p.b[0] = b0.x, p.b[1] = b0.y, p.b[2] = b1.x, p.b[3] = b1.y;
    }
    return p;
  }
};

template <int DT, bool VEC>
__device__ __forceinline__ void store_pairs(typename TrainElem<DT>::T* o, int c, int lg, int h, const Pairs& p) {
  if constexpr (VEC && DT == 2) {
    *reinterpret_cast<float4*>(o + 4 * c) = make_float4(p.a[0], p.a[1], p.a[2], p.a[3]);
    *reinterpret_cast<float4*>(o + 4 * c + h) = make_float4(p.b[0], p.b[1], p.b[2], p.b[3]);
  } else if constexpr (VEC) {
    using E = Elem<DT == 0>;
    *reinterpret_cast<uint2*>(o + 4 * c) = make_uint2(E::from_f2(p.a[0], p.a[1]), E::from_f2(p.a[2], p.a[3]));
    *reinterpret_cast<uint2*>(o + 4 * c + h) = make_uint2(E::from_f2(p.b[0], p.b[1]), E::from_f2(p.b[2], p.b[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = c + (j << lg);
      if (i < h) o[i] = TrainElem<DT>::from_f(p.a[j]), o[i + h] = TrainElem<DT>::from_f(p.b[j]);
    }
  }
}

template <bool VEC>
__device__ __forceinline__ Pairs load_table(const float* row, int c, int lg, int h) {
  RawPairs<2, VEC> t;
  t.load(row, c, lg, h);
  return t.get();
}

__device__ __forceinline__ float group_sum(float v, int lg) {
  for (int o = 1 << lg >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Blocks below side[0].blocks take the query heads, the others the key heads.  Item n of a
// side is the heads j per .. of row n / ranges, j = n % ranges; every group of a warp takes
// the same number of turns, those without a head left on zeros.
template <int DT, bool VEC, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? 2 : 3) head_norm_kernel(const __grid_constant__ HeadNormParams p) {
  using T = typename TrainElem<DT>::T;
  const bool second = blockIdx.x >= p.side[0].blocks;
  const HeadNormSide& sd = p.side[second];
  const unsigned block = blockIdx.x - (second ? p.side[0].blocks : 0u);
  const int lg = p.lg, c = threadIdx.x & ((1 << lg) - 1), h = p.D >> 1;
  const long long group = ((long long)block * kThreads + threadIdx.x) >> lg, lead = ((threadIdx.x & 31) >> lg);
  const long long groups = (long long)sd.blocks * kThreads >> lg;
  const int items = p.rows * sd.ranges;  // < 2^31, checked by the entry point

  Pairs w, acc;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = VEC ? 4 * c + j : c + (j << lg);
    auto weight = [&](int n) {
      return p.w32 ? static_cast<const float*>(sd.w)[n] : TrainElem<DT>::to_f(static_cast<const T*>(sd.w)[n]);
    };
    w.a[j] = i < h ? weight(i) : 0.f;
    w.b[j] = i < h ? weight(i + h) : 0.f;
    acc.a[j] = acc.b[j] = 0.f;
  }

  for (long long first = group - lead; first < items; first += groups) {
    const bool live = first + lead < items;
    const int item = (int)(live ? first + lead : 0), row = sd.by_ranges(item), head = (item - row * sd.ranges) * sd.per;
    const int b = p.by_s(row), s = row - b * p.S;
    const long long at = (p.start ? p.start[b] : 0) + (long long)s;
    const bool known = at >= 0 && at < p.cos_rows;
    if (live && !known && p.status) atomicExch(p.status, (int)kDevBadShape);
    Pairs cs{}, sn{};
    if (known) {
      cs = load_table<VEC>(p.cos + at * p.cs_stride, c, lg, h);
      sn = load_table<VEC>(p.sin + at * p.cs_stride, c, lg, h);
    }
    const int n = live ? min(sd.per, sd.heads - head) : 0;
    const T* x = static_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + head * sd.x_sh;
    T* o = static_cast<T*>(sd.out) + b * sd.o_sb + s * sd.o_ss + head * sd.o_sh;
    const T* g = BWD ? static_cast<const T*>(sd.grad) + b * sd.g_sb + s * sd.g_ss + head * sd.g_sh : nullptr;
    RawPairs<DT, VEC> nx{}, ng{};
    if (n > 0 && known) {
      nx.load(x, c, lg, h);
      if constexpr (BWD) ng.load(g, c, lg, h);
    }
    for (int k = 0; k < sd.per; ++k) {
      const Pairs v = nx.get();
      Pairs d;
      if constexpr (BWD) d = ng.get();
      const bool have = k < n;
      if (k + 1 < n && known) {
        x += sd.x_sh;
        nx.load(x, c, lg, h);
        if constexpr (BWD) {
          g += sd.g_sh;
          ng.load(g, c, lg, h);
        }
      }
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = fmaf(v.a[j], v.a[j], fmaf(v.b[j], v.b[j], ss));
      Pairs out;
      if constexpr (!BWD) {
        const float r = rsqrtf(fmaf(group_sum(ss, lg), p.inv_d, p.eps));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float ya = v.a[j] * r * w.a[j], yb = v.b[j] * r * w.b[j];
          out.a[j] = ya * cs.a[j] - yb * sn.a[j];
          out.b[j] = yb * cs.b[j] + ya * sn.b[j];
        }
      } else {
        float su = 0.f;
        Pairs dy;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dy.a[j] = d.a[j] * cs.a[j] + d.b[j] * sn.b[j];
          dy.b[j] = d.b[j] * cs.b[j] - d.a[j] * sn.a[j];
          su = fmaf(dy.a[j] * w.a[j], v.a[j], fmaf(dy.b[j] * w.b[j], v.b[j], su));
        }
        ss = group_sum(ss, lg);
        su = group_sum(su, lg);
        // A head that is not there adds nothing, whatever eps makes of its zeros.
        const float r = have && known ? rsqrtf(fmaf(ss, p.inv_d, p.eps)) : 0.f;
        const float m = su * r * r * p.inv_d;  // mean(u x^) r, to be multiplied with x
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc.a[j] = fmaf(dy.a[j], v.a[j] * r, acc.a[j]);
          acc.b[j] = fmaf(dy.b[j], v.b[j] * r, acc.b[j]);
          out.a[j] = r * (dy.a[j] * w.a[j] - v.a[j] * m);
          out.b[j] = r * (dy.b[j] * w.b[j] - v.b[j] * m);
        }
      }
      if (have) {
        if (!known) out = Pairs{};
        store_pairs<DT, VEC>(o, c, lg, h, out);
        o += sd.o_sh;
      }
    }
  }

  if constexpr (BWD) {
    // The block's sum, in a fixed order: lanes of the same place, then warps.
    __shared__ float sums[kThreads / 32][256];
    for (int o = 16; o >= 1 << lg; o >>= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc.a[j] += __shfl_xor_sync(0xffffffffu, acc.a[j], o);
        acc.b[j] += __shfl_xor_sync(0xffffffffu, acc.b[j], o);
      }
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) < 1 << lg)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = VEC ? 4 * c + j : c + (j << lg);
        if (i < h) sums[warp][i] = acc.a[j], sums[warp][i + h] = acc.b[j];
      }
    __syncthreads();
    if ((int)threadIdx.x < p.D) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) t += sums[k][threadIdx.x];
      if (sd.blocks > 1)
        sd.part[(long long)block * p.D + threadIdx.x] = t;
      else if (p.w32)
        static_cast<float*>(sd.dw)[threadIdx.x] = t;
      else
        static_cast<T*>(sd.dw)[threadIdx.x] = TrainElem<DT>::from_f(t);
    }
  }
}

// Adds the blocks' parts in a fixed order: block (x, y) columns 32 x .. of side y.
template <int DT>
__global__ void __launch_bounds__(1024) head_norm_sum_kernel(const __grid_constant__ HeadNormParams p) {
  __shared__ float sums[32][33];
  const HeadNormSide& sd = p.side[blockIdx.y];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < p.D && sd.blocks > 1)
    for (unsigned i = warp; i < sd.blocks; i += 32) t += sd.part[(long long)i * p.D + col];
  sums[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && col < p.D && sd.blocks > 1) {
    t = 0.f;
    for (int k = 0; k < 32; ++k) t += sums[k][lane];
    if (p.w32)
      static_cast<float*>(sd.dw)[col] = t;
    else
      static_cast<typename TrainElem<DT>::T*>(sd.dw)[col] = TrainElem<DT>::from_f(t);
  }
}

bool can_vector(const HeadNormParams& p, int dtype, bool bwd) {
  const long long step = 4;  // elements of an access
  const uintptr_t bytes = dtype == 2 ? 16 : 8;
  // Whole accesses, and a power of two of lanes.
  if (p.D % 8 || (p.D & (p.D - 1)) || p.cs_stride % 4 ||
      ((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15))
    return false;
  for (const HeadNormSide& s : p.side) {
    const void* ptrs[] = {s.x, s.out, bwd ? s.grad : nullptr};
    for (const void* q : ptrs)
      if (reinterpret_cast<uintptr_t>(q) % bytes) return false;
    const long long strides[] = {s.x_sb, s.x_ss, s.x_sh, s.o_sb, s.o_ss, s.o_sh,
                                 bwd ? s.g_sb : 0, bwd ? s.g_ss : 0, bwd ? s.g_sh : 0};
    for (long long q : strides)
      if (q % step) return false;
  }
  return true;
}

template <int DT, bool BWD>
cudaError_t launch(const HeadNormParams& p, bool vec, cudaStream_t st) {
  const unsigned grid = p.side[0].blocks + p.side[1].blocks;
  if (vec)
    head_norm_kernel<DT, true, BWD><<<grid, kThreads, 0, st>>>(p);
  else
    head_norm_kernel<DT, false, BWD><<<grid, kThreads, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (!BWD || e != cudaSuccess || (p.side[0].blocks == 1 && p.side[1].blocks == 1)) return e;
  head_norm_sum_kernel<DT><<<dim3((unsigned)(p.D + 31) / 32, 2), 1024, 0, st>>>(p);
  return cudaGetLastError();
}

int log_lanes(int D) {  // of the group that holds a head, four pairs a lane
  int lg = 0;
  while ((8 << lg) < D) ++lg;
  return lg;
}

}  // namespace

HeadNormSplit head_norm_split(long long rows, int heads, int other_heads, int D, bool bwd, int num_sms) {
  HeadNormSplit q;
  const int lg = log_lanes(D);
  const long long lanes = (long long)num_sms * 1024;  // that an SM holds of it
  const long long per = rows * heads / ((2 * lanes) >> lg);
  q.per = per < 1 ? 1 : per < heads ? (int)per : heads;
  q.ranges = (heads + q.per - 1) / q.per;
  q.per = (heads + q.ranges - 1) / q.ranges;
  const long long want = ((rows * q.ranges << lg) + kThreads - 1) / kThreads;
  long long cap = bwd ? (long long)num_sms * 2 * heads / (heads + other_heads) : (long long)num_sms * 32;
  if (cap < 1) cap = 1;
  q.blocks = (unsigned)(want < cap ? want : cap);
  return q;
}

cudaError_t launch_head_norm_sm100(HeadNormParams p, int dtype, bool bwd, cudaStream_t st) {
  p.lg = log_lanes(p.D);
  const bool vec = can_vector(p, dtype, bwd);
  if (dtype == 0) return bwd ? launch<0, true>(p, vec, st) : launch<0, false>(p, vec, st);
  if (dtype == 1) return bwd ? launch<1, true>(p, vec, st) : launch<1, false>(p, vec, st);
  return bwd ? launch<2, true>(p, vec, st) : launch<2, false>(p, vec, st);
}

}  // namespace dtk
