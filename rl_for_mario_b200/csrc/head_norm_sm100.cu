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
// one.  A head is held by a group of G lanes (a power of two), a few pairs (i, i + h) a lane,
// so that the rotation needs no exchange; the row sums are log2 G shuffles.  A group walks
// through some heads of one position with the position's table row in registers.
// 96 x 768 positions of 12 / 4 heads of 64, inputs cold: bf16 51 us forward (302 MB, 5.9
// TB/s) and 82 backward (453 MB, 5.5 TB/s), half the batch in fp32 47 and 70 (6.4 TB/s).  In
// 16 bits 55 % of the issue slots are in use, and most of what a warp waits for are loads from memory.
#include <type_traits>

#include "dt_common.cuh"
#include "dt_internal.h"
#include "train_common.cuh"

namespace dtk {

namespace {

constexpr int kThreads = 256;
// Blocks on an SM.  96 x 768, 12 / 4 heads of 64, bf16: forward 51 us with 3, 55 with 2, 76 with 4; backward 82 with 2, 96
// with 1, 193 with 3.  (With 2 the 16-bit gradients of 16-byte accesses spill 8 to 12 bytes a thread, those of single
// elements 12; nothing else does.)
template <bool BWD>
constexpr int kResident = BWD ? 2 : 3;

// ---------------------------------------------------------------- any width, stride and alignment
// Four pairs of a head as fp32: a[j], b[j] are elements i, i + h of pair i = c + G j of lane c; those at
// or past h read as 0 and are not written.
struct Pairs {
  float a[4], b[4];
};

// A head's elements as they stand in memory, on their way while another head is worked on.
template <int DT>
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
__device__ __forceinline__ void store_pairs(typename TrainElem<DT>::T* o, int c, int lg, int h, const Pairs& p) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = c + (j << lg);
    if (i < h) o[i] = TrainElem<DT>::from_f(p.a[j]), o[i + h] = TrainElem<DT>::from_f(p.b[j]);
  }
}

__device__ __forceinline__ Pairs load_table(const float* row, int c, int lg, int h) {
  RawPairs<2> t;
  t.load(row, c, lg, h);
  return t.get();
}

__device__ __forceinline__ float group_sum(float v, int lg) {
  for (int o = 1 << lg >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int LG>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1 << LG >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The block's part of a weight's gradient from its warps' [warps, D], in a fixed order.
template <int DT>
__device__ __forceinline__ void block_sum(const HeadNormParams& p, const HeadNormSide& sd, unsigned block,
                                          const float* sums) {
  __syncthreads();
  if ((int)threadIdx.x < p.D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) t += sums[k * p.D + threadIdx.x];
    if (sd.blocks > 1)
      sd.part[(long long)block * p.D + threadIdx.x] = t;
    else if (p.w32)
      static_cast<float*>(sd.dw)[threadIdx.x] = t;
    else
      static_cast<typename TrainElem<DT>::T*>(sd.dw)[threadIdx.x] = TrainElem<DT>::from_f(t);
  }
}

// Blocks below side[0].blocks take the query heads, the others the key heads.  Item n of a
// side is the heads `per` j .. of position n / ranges (all samples' in a row), j = n % ranges:
// neighbouring groups read neighbouring memory (with the same position of different samples
// side by side, which share a table row, 96 x 768, 12 / 4 heads of 64 took 66 us, 57 so).
// Every group of a warp takes the same number of turns, those without a head left on zeros.
struct Item {
  int b, s, head;
};
__device__ __forceinline__ Item item_of(const HeadNormParams& p, const HeadNormSide& sd, int item) {
  Item q;
  const int row = sd.by_ranges(item);
  q.head = (item - row * sd.ranges) * sd.per;
  q.b = p.by_s(row);
  q.s = row - q.b * p.S;
  return q;
}

template <int DT, bool BWD>
__global__ void __launch_bounds__(kThreads, kResident<BWD>) head_norm_any_kernel(const __grid_constant__ HeadNormParams p) {
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
    const int i = c + (j << lg);
    auto weight = [&](int n) {
      return p.w32 ? static_cast<const float*>(sd.w)[n] : TrainElem<DT>::to_f(static_cast<const T*>(sd.w)[n]);
    };
    w.a[j] = i < h ? weight(i) : 0.f;
    w.b[j] = i < h ? weight(i + h) : 0.f;
    acc.a[j] = acc.b[j] = 0.f;
  }

  for (long long first = group - lead; first < items; first += groups) {
    const bool live = first + lead < items;
    const Item it = item_of(p, sd, live ? (int)(first + lead) : 0);
    const int b = it.b, s = it.s, head = it.head;
    const long long at = (p.start ? p.start[b] : 0) + (long long)s;
    const bool known = at >= 0 && at < p.cos_rows;
    if (live && !known && p.status) atomicExch(p.status, (int)kDevBadShape);
    Pairs cs{}, sn{};
    if (known) {
      cs = load_table(p.cos + at * p.cs_stride, c, lg, h);
      sn = load_table(p.sin + at * p.cs_stride, c, lg, h);
    }
    const int n = live ? min(sd.per, sd.heads - head) : 0;
    const T* x = static_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + head * sd.x_sh;
    T* o = static_cast<T*>(sd.out) + b * sd.o_sb + s * sd.o_ss + head * sd.o_sh;
    const T* g = BWD ? static_cast<const T*>(sd.grad) + b * sd.g_sb + s * sd.g_ss + head * sd.g_sh : nullptr;
    RawPairs<DT> nx{}, ng{};
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
        store_pairs<DT>(o, c, lg, h, out);
        o += sd.o_sh;
      }
    }
  }

  if constexpr (BWD) {
    extern __shared__ float sums[];  // [warps, D]
    for (int o = 16; o >= 1 << lg; o >>= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc.a[j] += __shfl_xor_sync(0xffffffffu, acc.a[j], o);
        acc.b[j] += __shfl_xor_sync(0xffffffffu, acc.b[j], o);
      }
    float* mine = sums + (threadIdx.x >> 5) * p.D;
    if ((threadIdx.x & 31) < 1 << lg)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = c + (j << lg);
        if (i < h) mine[i] = acc.a[j], mine[i + h] = acc.b[j];
      }
    block_sum<DT>(p, sd, block, sums);
  }
}

// ---------------------------------------------------------------- heads of whole vectors
// Lane c of a group holds elements P c .. P c + P - 1 and the same from h on: two accesses of 16 bytes
// (P = 8, fp32 4), or of 8 for 16-bit heads whose halves are not whole 16-byte vectors (P = 4).  A head's elements are copied into the lane's own places of a ring in shared memory,
// kDepth heads ahead and across positions, and only the lane reads them back: no barrier, and what is in
// flight takes no registers (one head ahead in registers: 107 + 178 us at 96 x 768, 12 / 4 heads of 64, bf16, when a
// first ring took 66 + 99).  Two heads ahead: 51 + 82 us there, half the batch in fp32 47 + 70; one 59 + 86 and 51 + 80;
// three and four 51 + 82 and 47 + 72.
template <int DT, int P>
using Vec = typename std::conditional<P * (DT == 2 ? 4 : 2) == 16, uint4, uint2>::type;
constexpr int kDepth = 2;

template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_vec(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}
__device__ __forceinline__ void copy_vec(uint2* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}

// A lane's half of a head as packed pairs of fp32.
template <int DT, int P>
struct Half {
  float2 p[P / 2];
  __device__ __forceinline__ void set(uint4 u) {
    if constexpr (DT == 2) {
      p[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
      p[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
    } else {
      using E = Elem<DT == 0>;
      p[0] = E::to_f2(u.x), p[1] = E::to_f2(u.y), p[P / 2 - 2] = E::to_f2(u.z), p[P / 2 - 1] = E::to_f2(u.w);
    }
  }
  __device__ __forceinline__ void set(uint2 u) {
    using E = Elem<DT == 0>;
    p[0] = E::to_f2(u.x), p[1] = E::to_f2(u.y);
  }
  __device__ __forceinline__ Vec<DT, P> bits() const {
    if constexpr (DT == 2) {
      return make_uint4(__float_as_uint(p[0].x), __float_as_uint(p[0].y), __float_as_uint(p[1].x),
                        __float_as_uint(p[1].y));
    } else {
      using E = Elem<DT == 0>;
      if constexpr (P == 4)
        return make_uint2(E::from_f2(p[0].x, p[0].y), E::from_f2(p[1].x, p[1].y));
      else
        return make_uint4(E::from_f2(p[0].x, p[0].y), E::from_f2(p[1].x, p[1].y), E::from_f2(p[2].x, p[2].y),
                          E::from_f2(p[3].x, p[3].y));
    }
  }
  __device__ __forceinline__ void load_f32(const float* f) {
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(f + 4 * i);
      p[2 * i] = make_float2(v.x, v.y);
      p[2 * i + 1] = make_float2(v.z, v.w);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) p[i] = make_float2(0.f, 0.f);
  }
};
__device__ __forceinline__ float2 minus(float2 v) { return make_float2(-v.x, -v.y); }

// Where a group stands in its walk: the heads of its items, one after the other.
template <typename T>
struct Place {
  const T* x;
  const T* g;
  int k, n;  // n: heads of the item, 0 behind the last one
};

template <int DT, int P, bool BWD, int LG>
__global__ void __launch_bounds__(kThreads, kResident<BWD>) head_norm_kernel(const __grid_constant__ HeadNormParams p) {
  using T = typename TrainElem<DT>::T;
  using V = Vec<DT, P>;
  constexpr int N = P / 2, TENSORS = BWD ? 4 : 2;
  extern __shared__ uint4 ring_bytes[];
  V* ring = reinterpret_cast<V*>(ring_bytes);  // [kDepth, TENSORS, threads]
  __shared__ __align__(16) float weights[256];
  const bool second = blockIdx.x >= p.side[0].blocks;
  const HeadNormSide& sd = p.side[second];
  const unsigned block = blockIdx.x - (second ? p.side[0].blocks : 0u);
  constexpr int lg = LG;
  const int c = threadIdx.x & ((1 << lg) - 1), h = p.D >> 1;
  const bool mine = c * P < h;
  const int e = mine ? c * P : 0;  // the lane's first element
  for (int i = threadIdx.x; i < p.D; i += kThreads)
    weights[i] = p.w32 ? static_cast<const float*>(sd.w)[i] : TrainElem<DT>::to_f(static_cast<const T*>(sd.w)[i]);
  __syncthreads();
  const long long items = (long long)p.rows * sd.ranges;
  const long long groups = (long long)sd.blocks * kThreads >> lg;
  const long long group = ((long long)block * kThreads + threadIdx.x) >> lg, lead = (threadIdx.x & 31) >> lg;

  // (Items number less than 2^31; a warp's groups take the same number of turns.)
  long long at = group - lead;  // the warp's first item of the turn that is copied
  Place<T> f;
  auto enter = [&](Place<T>& q, long long first) {
    const bool live = first + lead < items;
    const Item it = item_of(p, sd, live ? (int)(first + lead) : 0);
    q.n = live && mine ? min(sd.per, sd.heads - it.head) : 0;
    q.k = 0;
    q.x = static_cast<const T*>(sd.x) + it.b * sd.x_sb + it.s * sd.x_ss + it.head * sd.x_sh + e;
    if constexpr (BWD) q.g = static_cast<const T*>(sd.grad) + it.b * sd.g_sb + it.s * sd.g_ss + it.head * sd.g_sh + e;
  };
  V* slots = ring + threadIdx.x;
  auto fetch = [&](int stage) {
    if (f.k < f.n) {
      V* to = slots + stage * (TENSORS * kThreads);
      copy_vec(to, f.x);
      copy_vec(to + kThreads, f.x + h);
      if constexpr (BWD) {
        copy_vec(to + 2 * kThreads, f.g);
        copy_vec(to + 3 * kThreads, f.g + h);
      }
    }
    copies_commit();
    f.x += sd.x_sh;
    if constexpr (BWD) f.g += sd.g_sh;
    if (++f.k == sd.per && at + groups < items) {
      at += groups;
      enter(f, at);
    }
  };
  Half<DT, P> aa, ab;  // sums of the weight's gradient
  aa.clear();
  ab.clear();
  if (at < items) {
    enter(f, at);
#pragma unroll
    for (int i = 0; i < kDepth; ++i) fetch(i);
  }
  int stage = 0;
  for (long long first = group - lead; first < items; first += groups) {
    const bool live = first + lead < items;
    const Item it = item_of(p, sd, live ? (int)(first + lead) : 0);
    const int b = it.b, s = it.s, head = it.head;
    const int n = live && mine ? min(sd.per, sd.heads - head) : 0;
    T* o = static_cast<T*>(sd.out) + b * sd.o_sb + s * sd.o_ss + head * sd.o_sh + e;
    const long long t = (p.start ? p.start[b] : 0) + (long long)s;
    const bool known = t >= 0 && t < p.cos_rows;
    if (live && !known && p.status) atomicExch(p.status, (int)kDevBadShape);
    Half<DT, P> ca, cb, sa, sb;  // forward: times the weights
    const float* cos = p.cos + (known ? t : 0) * p.cs_stride + e;
    const float* sin = p.sin + (known ? t : 0) * p.cs_stride + e;
    ca.load_f32(cos), cb.load_f32(cos + h), sa.load_f32(sin), sb.load_f32(sin + h);
    if constexpr (!BWD) {
      Half<DT, P> wa, wb;
      wa.load_f32(weights + e), wb.load_f32(weights + e + h);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        ca.p[i] = fmul2(ca.p[i], wa.p[i]), cb.p[i] = fmul2(cb.p[i], wb.p[i]);
        sa.p[i] = minus(fmul2(sa.p[i], wb.p[i])), sb.p[i] = fmul2(sb.p[i], wa.p[i]);
      }
    }
    for (int k = 0; k < sd.per; ++k) {
      copies_wait<kDepth - 1>();
      const V* from = slots + stage * (TENSORS * kThreads);
      const bool have = k < n;
      const V zero{};
      Half<DT, P> xa, xb, ga, gb;
      xa.set(have ? from[0] : zero), xb.set(have ? from[kThreads] : zero);
      if constexpr (BWD) ga.set(have ? from[2 * kThreads] : zero), gb.set(have ? from[3 * kThreads] : zero);
      fetch(stage);
      stage = stage + 1 == kDepth ? 0 : stage + 1;
      float2 q = make_float2(0.f, 0.f), z = q;
#pragma unroll
      for (int i = 0; i < N; ++i) q = ffma2(xa.p[i], xa.p[i], ffma2(xb.p[i], xb.p[i], q));
      if constexpr (!BWD) {
        const float r = rsqrtf(fmaf(group_sum<LG>(both_sum(q)), p.inv_d, p.eps));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float2 a = xa.p[i], v = xb.p[i];
          xa.p[i] = fmul2(ffma2(v, sa.p[i], fmul2(a, ca.p[i])), both(r));
          xb.p[i] = fmul2(ffma2(a, sb.p[i], fmul2(v, cb.p[i])), both(r));
        }
      } else {
        Half<DT, P> wa, wb;
        wa.load_f32(weights + e), wb.load_f32(weights + e + h);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float2 a = ga.p[i], v = gb.p[i];
          ga.p[i] = ffma2(v, sb.p[i], fmul2(a, ca.p[i]));
          gb.p[i] = ffma2(minus(a), sa.p[i], fmul2(v, cb.p[i]));
          wa.p[i] = fmul2(ga.p[i], wa.p[i]);
          wb.p[i] = fmul2(gb.p[i], wb.p[i]);
          z = ffma2(wa.p[i], xa.p[i], ffma2(wb.p[i], xb.p[i], z));
        }
        const float ss = group_sum<LG>(both_sum(q)), su = group_sum<LG>(both_sum(z));
        // A head that is not there adds nothing, whatever eps makes of its zeros.
        const float r = have && known ? rsqrtf(fmaf(ss, p.inv_d, p.eps)) : 0.f;
        const float m = -su * r * r * p.inv_d;  // - mean(u x^) r, to be multiplied with x
#pragma unroll
        for (int i = 0; i < N; ++i) {
          aa.p[i] = ffma2(ga.p[i], fmul2(xa.p[i], both(r)), aa.p[i]);
          ab.p[i] = ffma2(gb.p[i], fmul2(xb.p[i], both(r)), ab.p[i]);
          xa.p[i] = fmul2(ffma2(xa.p[i], both(m), wa.p[i]), both(r));
          xb.p[i] = fmul2(ffma2(xb.p[i], both(m), wb.p[i]), both(r));
        }
      }
      if (have) {
        *reinterpret_cast<V*>(o) = known ? xa.bits() : zero;
        *reinterpret_cast<V*>(o + h) = known ? xb.bits() : zero;
        o += sd.o_sh;
      }
    }
  }
  copies_wait<0>();

  if constexpr (BWD) {
    __syncthreads();  // (the ring's last readers are done)
    float* sums = reinterpret_cast<float*>(ring_bytes);  // [warps, D]
#pragma unroll
    for (int o = 16; o >= 1 << lg; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        aa.p[i].x += __shfl_xor_sync(0xffffffffu, aa.p[i].x, o), aa.p[i].y += __shfl_xor_sync(0xffffffffu, aa.p[i].y, o);
        ab.p[i].x += __shfl_xor_sync(0xffffffffu, ab.p[i].x, o), ab.p[i].y += __shfl_xor_sync(0xffffffffu, ab.p[i].y, o);
      }
    float* row = sums + (threadIdx.x >> 5) * p.D + e;
    if ((threadIdx.x & 31) < 1 << lg && mine)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        *reinterpret_cast<float2*>(row + 2 * i) = aa.p[i];
        *reinterpret_cast<float2*>(row + h + 2 * i) = ab.p[i];
      }
    block_sum<DT>(p, sd, block, sums);
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

// Elements of an access of the vector kernel: every half of a head has to be whole vectors on boundaries of their size.
// 0: there is no such size.  (96 x 768, 8 / 2 heads of 40, bf16: 45 + 73 us with accesses of 8 bytes, 82 + 124 element by
// element.)
int vector_pairs(const HeadNormParams& p, int dtype, bool bwd) {
  if (p.cs_stride % 4 || ((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15)) return 0;
  for (int pairs = dtype == 2 ? 4 : 8; pairs >= 4; pairs /= 2) {
    const uintptr_t bytes = (uintptr_t)pairs * (dtype == 2 ? 4 : 2);
    bool fits = p.D % (2 * pairs) == 0;
    for (const HeadNormSide& s : p.side) {
      const void* ptrs[] = {s.x, s.out, bwd ? s.grad : nullptr};
      for (const void* q : ptrs) fits = fits && reinterpret_cast<uintptr_t>(q) % bytes == 0;
      const long long strides[] = {s.x_sb, s.x_ss, s.x_sh, s.o_sb, s.o_ss, s.o_sh,
                                   bwd ? s.g_sb : 0, bwd ? s.g_ss : 0, bwd ? s.g_sh : 0};
      for (long long q : strides) fits = fits && q % pairs == 0;
    }
    if (fits) return pairs;
  }
  return 0;
}

int log_lanes(int D, int pairs) {  // of the group that holds a head
  int lg = 0;
  while ((2 * pairs << lg) < D) ++lg;
  return lg;
}

template <int DT, int P, bool BWD>
cudaError_t launch_vector(const HeadNormParams& p, unsigned grid, cudaStream_t st) {
  constexpr int ring = kDepth * (BWD ? 4 : 2) * kThreads * (int)sizeof(Vec<DT, P>), sums = kThreads / 32 * 256 * 4;
  constexpr int smem = BWD && sums > ring ? sums : ring;  // (the block's sums lie in the ring)
  auto run = [&](auto kernel) {
    const cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kernel), smem);
    if (e == cudaSuccess) kernel<<<grid, kThreads, smem, st>>>(p);
    return e;
  };
  switch (p.lg) {
    case 0: return run(head_norm_kernel<DT, P, BWD, 0>);
    case 1: return run(head_norm_kernel<DT, P, BWD, 1>);
    case 2: return run(head_norm_kernel<DT, P, BWD, 2>);
    case 3: return run(head_norm_kernel<DT, P, BWD, 3>);
    case 4: return run(head_norm_kernel<DT, P, BWD, 4>);
    case 5: return run(head_norm_kernel<DT, P, BWD, 5>);
  }
  return cudaErrorInvalidValue;
}

template <int DT, bool BWD>
cudaError_t launch(const HeadNormParams& p, cudaStream_t st) {
  const unsigned grid = p.side[0].blocks + p.side[1].blocks;
  cudaError_t e = cudaSuccess;
  if (p.vec == 8) {
    if constexpr (DT != 2) e = launch_vector<DT, 8, BWD>(p, grid, st);
  } else if (p.vec == 4) {
    e = launch_vector<DT, 4, BWD>(p, grid, st);
  } else {
    head_norm_any_kernel<DT, BWD><<<grid, kThreads, BWD ? kThreads / 32 * p.D * 4 : 0, st>>>(p);
  }
  if (e == cudaSuccess) e = cudaGetLastError();
  if (!BWD || e != cudaSuccess || (p.side[0].blocks == 1 && p.side[1].blocks == 1)) return e;
  head_norm_sum_kernel<DT><<<dim3((unsigned)(p.D + 31) / 32, 2), 1024, 0, st>>>(p);
  return cudaGetLastError();
}

struct Split {
  int per, ranges;
  unsigned blocks;
};

// How a side's heads are spread: blocks in proportion to them, as many as the GPU holds at a time, and each
// position's heads cut into the number of ranges that takes a group the least time: turns of (heads of a
// range + 1), the start of an item (table row, weights) costing about as much as a head.
Split split_heads(long long rows, int heads, int other_heads, int D, int pairs, bool bwd, int num_sms) {
  const int lg = log_lanes(D, pairs);
  long long cap = (long long)num_sms * (bwd ? kResident<true> : kResident<false>) * heads / (heads + other_heads);
  if (cap < 1) cap = 1;
  const long long groups = cap * kThreads >> lg;
  Split q{heads, 1, 1u};
  long long best = -1;
  for (int ranges = 1; ranges <= heads; ++ranges) {
    const int per = (heads + ranges - 1) / ranges;
    if ((long long)(ranges - 1) * per >= heads) continue;  // the last would be empty
    const long long cost = (rows * ranges + groups - 1) / groups * (per + 1);
    if (best < 0 || cost < best) best = cost, q.per = per, q.ranges = ranges;
  }
  const long long want = ((rows * q.ranges << lg) + kThreads - 1) / kThreads;
  q.blocks = (unsigned)(want < cap ? want : cap);
  return q;
}

}  // namespace

void head_norm_plan(HeadNormParams& p, int dtype, bool bwd, int num_sms) {
  p.vec = vector_pairs(p, dtype, bwd);
  const int pairs = p.vec ? p.vec : 4;
  p.lg = log_lanes(p.D, pairs);
  for (int i = 0; i < 2; ++i) {
    HeadNormSide& s = p.side[i];
    const Split q = split_heads(p.rows, s.heads, p.side[1 - i].heads, p.D, pairs, bwd, num_sms);
    s.per = q.per, s.ranges = q.ranges, s.blocks = q.blocks, s.by_ranges = FastDiv((uint32_t)q.ranges);
  }
}

// Alignment decides between two plans when the backward call comes: room for either.
long long head_norm_parts(long long rows, int Hq, int Hkv, int D, int num_sms) {
  long long most = 0;
  for (int pairs = 4; pairs <= 8; pairs += 4) {
    const long long n = (long long)split_heads(rows, Hq, Hkv, D, pairs, true, num_sms).blocks +
                        split_heads(rows, Hkv, Hq, D, pairs, true, num_sms).blocks;
    most = n > most ? n : most;
  }
  return most;
}

cudaError_t launch_head_norm_sm100(const HeadNormParams& p, int dtype, bool bwd, cudaStream_t st) {
  if (dtype == 0) return bwd ? launch<0, true>(p, st) : launch<0, false>(p, st);
  if (dtype == 1) return bwd ? launch<1, true>(p, st) : launch<1, false>(p, st);
  return bwd ? launch<2, true>(p, st) : launch<2, false>(p, st);
}

}  // namespace dtk
