// The end of a training step over all of a model's tensors at once: the norm of the
// gradient and the AdamW update (Loshchilov, Hutter, ICLR 2019), clipped by it.
//
//   c = min(1, max_norm / (norm + 1e-6)),  g' = c g
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)      t the step, from 1
//
// Tensors are cut into blocks of 256 elements, a warp's work; a tensor starts a new block, so
// the averages of tensor i lie from element 256 (blocks before it) on in flat arrays of whole
// blocks.  Pointers and sizes travel as kernel arguments (up to 960 tensors a launch): there
// is no table on the device to be built, kept or to go stale.
//
// Averages in 8 bits: a block of each shares a scale 2^e, e from its largest value.  m is kept as
// sign, four exponent and three further bits, v, which has no sign, as five exponent and three
// further bits (the upper bits of a half number).  Two things make so few bits serve an average:
//  - Rounding is up or down at random, by the part cut off (words of the Philox generator of
//    philox.cuh, a function of seed, step and element), so that a change of v by 0.1 % of the way
//    to g^2, less than a hundredth of the spacing, happens once in so many steps instead of never.
//  - The scale is a power of two, so that a value that stays put is stored exactly while the
//    block's largest changes: the random rounding then only sees the change.  With values off the grid
//    every step would add the variance of a full rounding, spacing^2 / 6, and v with its memory
//    of 1 / (1 - b2) = 1,000 steps would carry noise of 80 % of itself; so it is about 20 %, 10 % in its root.
// A v above zero never becomes zero, so that no m is divided by eps alone.
//
// Bound by HBM: bytes an element, bf16 weights: 22 with 32-bit averages, 10 with 8-bit ones, 28 with
// fp32 weights beside them.
#include <cstring>

#include "dt_common.cuh"
#include "dt_internal.h"
#include "philox.cuh"
#include "train_common.cuh"

namespace dtk {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kNormUnit = 1024;      // elements of a warp's turn in the norm
constexpr uint32_t kSite = 0xffffffffu;  // the generator's site of the averages' rounding
constexpr int kMinScale = 32;        // exponents of scales (biased): their products with any code are normal numbers

template <int N>
struct TensorTable {
  TensorSlot slot[N];
};

// The slot that holds unit b: the number of slots that end at or before it.
__device__ __forceinline__ int find_slot(const uint32_t* ends, int count, uint32_t b, int lane) {
  int t = 0;
  for (int i = 0; i < count; i += 32) {
    const bool before = i + lane < count && ends[i + lane] <= b;
    const unsigned m = __ballot_sync(0xffffffffu, before);
    t += __popc(m);
    if (m != 0xffffffffu) break;
  }
  return t;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<unsigned long long>(p) & 15) == 0; }

// Eight elements from `at` on of a tensor of element code DT; those past its end read as 0 and are not written.
template <int DT>
__device__ __forceinline__ void get8(const void* base, long long at, long long n, bool vec, float (&v)[8]) {
  using T = typename TrainElem<DT>::T;
  const T* x = static_cast<const T*>(base) + at;
  if (vec && at + 8 <= n) {
    load8<DT, true>(x, 0, 0, 8, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i < n ? TrainElem<DT>::to_f(x[i]) : 0.f;
  }
}
template <int DT>
__device__ __forceinline__ void put8(void* base, long long at, long long n, bool vec, const float (&v)[8]) {
  using T = typename TrainElem<DT>::T;
  T* x = static_cast<T*>(base) + at;
  if (vec && at + 8 <= n) {
    store8<DT, true>(x, 0, 0, 8, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < n) x[i] = TrainElem<DT>::from_f(v[i]);
  }
}
// By the tensor's own code (the same for a warp).
__device__ __forceinline__ void get8_of(int code, const void* base, long long at, long long n, bool vec, float (&v)[8]) {
  if (code == 0) get8<0>(base, at, n, vec, v);
  else if (code == 1) get8<1>(base, at, n, vec, v);
  else get8<2>(base, at, n, vec, v);
}
__device__ __forceinline__ void put8_of(int code, void* base, long long at, long long n, bool vec, const float (&v)[8]) {
  if (code == 0) put8<0>(base, at, n, vec, v);
  else if (code == 1) put8<1>(base, at, n, vec, v);
  else put8<2>(base, at, n, vec, v);
}

// The block's sum of a value of each thread, in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) v += red[i];
  return v;
}

// ---------------------------------------------------------------- norm
// Sums of eight squares are fp32 where that loses nothing, else fp64 (squares of numbers
// beyond 2^63 overflow in fp32, those of numbers below 2^-63 lose their bits); sums of
// those fp64.
__device__ __forceinline__ double square8(const float (&v)[8]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(v[i], v[i], s);
  if (s >= 1e-28f && s <= 1e38f) return (double)s;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) d += (double)v[i] * (double)v[i];
  return d;
}

template <int N>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ TensorTable<N> table,
                                                             const __grid_constant__ GradNormParams p) {
  __shared__ uint32_t ends[N];
  __shared__ double red[kWarps];
  for (int i = threadIdx.x; i < p.count; i += kThreads) ends[i] = table.slot[i].end;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  for (uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < p.units; u += gridDim.x * kWarps) {
    const int t = find_slot(ends, p.count, u, lane);
    const TensorSlot& s = table.slot[t];
    if (!s.g) continue;
    const long long first = (long long)(u - (t ? ends[t - 1] : 0u)) * kNormUnit + lane * 8;
    const bool vec = aligned16(s.g);
#pragma unroll
    for (int i = 0; i < kNormUnit / 256; ++i) {
      float v[8];
      get8_of(s.kind & 3, s.g, first + i * 256, s.n, vec, v);
      sum += square8(v);
    }
  }
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) {
    if (p.norm)
      *p.norm = (float)sqrt(sum);
    else
      p.parts[blockIdx.x] = sum;
  }
}

__device__ __forceinline__ double sum_parts(const double* parts, int n, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v += parts[i];
  return block_sum(v, red);
}

__global__ void __launch_bounds__(kThreads) grad_norm_sum_kernel(const double* parts, int n, float* norm) {
  __shared__ double red[kWarps];
  const double s = sum_parts(parts, n, red);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// ---------------------------------------------------------------- averages in 8 bits
__device__ __forceinline__ float scale_of(int field) { return __uint_as_float((uint32_t)field << 23); }

// What codes of a block are multiplied with; a block that met a value that is not finite is one of NaNs.
template <int TOP>
__device__ __forceinline__ float decode_scale(int e) {
  return e == 255 ? __uint_as_float(0x7fc00000u) : scale_of(max(e, kMinScale) - TOP);
}

// Four codes of the first (second) average as fp32, without their block's scale.
__device__ __forceinline__ void decode_first(uint32_t codes, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)(codes >> (16 * i))));
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void decode_second(uint32_t codes, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // Two codes, each 7 bits up in a half of its own.
    uint32_t h = __byte_perm(codes, 0, i ? 0x4342 : 0x4140) << 7;
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// y >= 0, scaled into the codes' range (2^(TOP + 1) at most), rounded up or down by u, a 16-bit word:
// three bits behind the leading one, from 2^(1 - BIAS) down in steps of 2^(-2 - BIAS).
template <int BIAS>
__device__ __forceinline__ uint32_t encode(float y, uint32_t u) {
  const uint32_t small = ((uint32_t)__float2int_rz(y * (float)(1ull << (BIAS + 18))) + u) >> 16;
  const uint32_t large = ((__float_as_uint(y) + (u << 4)) >> 20) - ((127u - BIAS) << 3);
  return y < 1.f / (1 << (BIAS - 1)) ? small : large;
}

// Stores a lane's eight values of a block; returns nothing, the block's scale goes with lane 0.
template <int BIAS, int TOP, bool SIGNED>
__device__ __forceinline__ void put_codes(uint8_t* codes, uint8_t* scale, const float (&x)[8], const uint4& words, int lane) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
  const int e = max((int)(__reduce_max_sync(0xffffffffu, most) >> 23), kMinScale);
  const float f = scale_of(254 + TOP - min(e, 254));
  const uint32_t w[4] = {words.x, words.y, words.z, words.w};
  uint32_t c[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    uint32_t k = encode<BIAS>(fabsf(x[i]) * f, u) & 0xffu;
    if constexpr (SIGNED)
      k |= __float_as_uint(x[i]) >> 24 & 0x80u;
    else
      k = x[i] > 0.f ? max(k, 1u) : k;
    c[i >> 2] |= k << (8 * (i & 3));
  }
  *reinterpret_cast<uint2*>(codes) = make_uint2(c[0], c[1]);
  if (lane == 0) *scale = (uint8_t)e;
}

// ---------------------------------------------------------------- step
struct GroupNow {
  float rate, root, decay, b1, c1, b2, c2, eps;
};

// Off by an ulp at most; the weights' own rounding is larger than what it does to a step.
__device__ __forceinline__ float fast_sqrt(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// x^n by squaring.
__device__ __forceinline__ double power(double x, unsigned long long n) {
  double r = 1.0;
  for (; n; n >>= 1, x *= x)
    if (n & 1) r *= x;
  return r;
}

template <bool BITS8, int N>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ TensorTable<N> table,
                                                            const __grid_constant__ AdamWParams p) {
  __shared__ uint32_t ends[N];
  __shared__ GroupNow groups[kAdamWGroups];
  __shared__ double red[kWarps];
  const long long seed = p.state[0], step = p.state[1] + 1;
  if ((int)threadIdx.x < p.ngroups) {
    const AdamWGroup& q = p.group[threadIdx.x];
    const double lr = q.lr_ptr ? (double)*q.lr_ptr : q.lr;
    const double k1 = 1.0 - power(q.b1, step), k2 = 1.0 - power(q.b2, step);
    groups[threadIdx.x] = GroupNow{(float)(lr / k1),  (float)(1.0 / sqrt(k2)),  (float)(1.0 - lr * q.wd),
                                   (float)q.b1,       (float)(1.0 - q.b1),      (float)q.b2,
                                   (float)(1.0 - q.b2), (float)q.eps};
  }
  for (int i = threadIdx.x; i < p.count; i += kThreads) ends[i] = table.slot[i].end;
  float clip = 1.f;
  bool skip = false;
  if (p.parts) {
    const float norm = (float)sqrt(sum_parts(p.parts, p.nparts, red));
    clip = fminf(1.f, __fdiv_rn(p.max_norm, __fadd_rn(norm, 1e-6f)));
    skip = !isfinite(norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.norm = norm;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const DropKey key{(uint32_t)seed, (uint32_t)((unsigned long long)seed >> 32), (uint32_t)step, kSite};
  if (!skip)
    for (uint32_t b = blockIdx.x * kWarps + (threadIdx.x >> 5); b < p.units; b += gridDim.x * kWarps) {
      const int t = find_slot(ends, p.count, b, lane);
      const TensorSlot& s = table.slot[t];
      if (!s.g) continue;
      const int code = s.kind & 3;
      const GroupNow& q = groups[s.kind >> 8];
      const long long n = s.n, at = (long long)(b - (t ? ends[t - 1] : 0u)) * 256 + lane * 8;
      const long long block = p.first + b, mine = block * 256 + lane * 8;
      const bool vec_p = aligned16(s.p), vec_g = aligned16(s.g), master = p.master && code != 2;
      float w[8], g[8], m[8], v[8];
      get8_of(code, s.g, at, n, vec_g, g);
      if (master)
        load8<2, true>(p.master + mine, 0, 0, 8, w);
      else
        get8_of(code, s.p, at, n, vec_p, w);
      if constexpr (BITS8) {
        const uint2 cm = *reinterpret_cast<const uint2*>(static_cast<uint8_t*>(p.m) + mine);
        const uint2 cv = *reinterpret_cast<const uint2*>(static_cast<uint8_t*>(p.v) + mine);
        const float fm = decode_scale<7>(p.m_scale[block]), fv = decode_scale<14>(p.v_scale[block]);
        decode_first(cm.x, m), decode_first(cm.y, m + 4);
        decode_second(cv.x, v), decode_second(cv.y, v + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] *= fm, v[i] *= fv;
      } else {
        load8<2, true>(static_cast<float*>(p.m) + mine, 0, 0, 8, m);
        load8<2, true>(static_cast<float*>(p.v) + mine, 0, 0, 8, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // Each product and sum of the averages rounded by itself: what is stored does not depend on how a
        // compiler contracts them.
        const float h = __fmul_rn(g[i], clip);
        m[i] = __fadd_rn(__fmul_rn(m[i], q.b1), __fmul_rn(h, q.c1));
        v[i] = __fadd_rn(__fmul_rn(v[i], q.b2), __fmul_rn(__fmul_rn(h, h), q.c2));
        w[i] = w[i] * q.decay - q.rate * __fdividef(m[i], fmaf(fast_sqrt(v[i]), q.root, q.eps));
      }
      if (master) store8<2, true>(p.master + mine, 0, 0, 8, w);
      put8_of(code, s.p, at, n, vec_p, w);
      if constexpr (BITS8) {
        const uint4 u = philox7(key, (unsigned long long)block * 32 + lane);
        // One word for both averages, its bytes turned over for the first.
        const uint4 r = make_uint4(__byte_perm(u.x, 0, 0x2301), __byte_perm(u.y, 0, 0x2301),
                                   __byte_perm(u.z, 0, 0x2301), __byte_perm(u.w, 0, 0x2301));
        put_codes<7, 7, true>(static_cast<uint8_t*>(p.m) + mine, p.m_scale + block, m, r, lane);
        put_codes<15, 14, false>(static_cast<uint8_t*>(p.v) + mine, p.v_scale + block, v, u, lane);
      } else {
        store8<2, true>(static_cast<float*>(p.m) + mine, 0, 0, 8, m);
        store8<2, true>(static_cast<float*>(p.v) + mine, 0, 0, 8, v);
      }
    }
  // The last block to come here counts the step; every block has read it by then.
  if (threadIdx.x == 0 && p.ticket && !skip) {
    __threadfence();
    if (atomicAdd(p.ticket, 1u) == gridDim.x - 1) {
      *p.ticket = 0u;
      p.state[1] = step;
    }
  }
}

// The averages as the numbers that their codes stand for, which bf16 holds exactly.
__global__ void __launch_bounds__(kThreads) adamw_moments_kernel(const uint8_t* m, const uint8_t* m_scale, const uint8_t* v,
                                                                 const uint8_t* v_scale, long long blocks,
                                                                 __nv_bfloat16* m_out, __nv_bfloat16* v_out) {
  const int lane = threadIdx.x & 31;
  for (long long b = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); b < blocks; b += (long long)gridDim.x * kWarps) {
    const long long at = b * 256 + lane * 8;
    const uint2 cm = *reinterpret_cast<const uint2*>(m + at), cv = *reinterpret_cast<const uint2*>(v + at);
    const float fm = decode_scale<7>(m_scale[b]), fv = decode_scale<14>(v_scale[b]);
    float x[8], y[8];
    decode_first(cm.x, x), decode_first(cm.y, x + 4);
    decode_second(cv.x, y), decode_second(cv.y, y + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= fm, y[i] *= fv;
    store8<0, true>(m_out + at, 0, 0, 8, x);
    store8<0, true>(v_out + at, 0, 0, 8, y);
  }
}

// Lengths of the argument list: a launch copies all of it.
constexpr int kFew = 64, kSome = 192;

// Calls f with the shortest list that holds the tensors.
template <int N, typename F>
void with_table(const TensorSlot* slots, int count, F f) {
  TensorTable<N> t;
  memcpy(t.slot, slots, sizeof(TensorSlot) * (size_t)count);
  f(t);
}
template <typename F>
void with_tables(const TensorSlot* slots, int count, F f) {
  if (count <= kFew) with_table<kFew>(slots, count, f);
  else if (count <= kSome) with_table<kSome>(slots, count, f);
  else with_table<kMaxTensors>(slots, count, f);
}

unsigned grid_for(long long units, int num_sms, int resident) {
  const long long want = (units + kWarps - 1) / kWarps, cap = (long long)num_sms * resident;
  return (unsigned)(want < 1 ? 1 : want < cap ? want : cap);
}

}  // namespace

constexpr int kNormResident = 8, kStepResident = 4;

int grad_norm_grid(long long units, int num_sms) { return (int)grid_for(units, num_sms, kNormResident); }
long long grad_norm_unit() { return kNormUnit; }

cudaError_t launch_grad_norm_sm100(const TensorSlot* slots, const GradNormParams& p, int num_sms, cudaStream_t st) {
  const unsigned grid = (unsigned)grad_norm_grid(p.units, num_sms);
  with_tables(slots, p.count, [&](const auto& t) {
    grad_norm_kernel<<<grid, kThreads, 0, st>>>(t, p);
  });
  return cudaGetLastError();
}

cudaError_t launch_grad_norm_sum_sm100(const double* parts, int n, float* norm, cudaStream_t st) {
  grad_norm_sum_kernel<<<1, kThreads, 0, st>>>(parts, n, norm);
  return cudaGetLastError();
}

cudaError_t launch_adamw_sm100(const TensorSlot* slots, const AdamWParams& p, int num_sms, cudaStream_t st) {
  const unsigned grid = grid_for(p.units, num_sms, kStepResident);
  with_tables(slots, p.count, [&](const auto& t) {
    if (p.m_scale)
      adamw_kernel<true><<<grid, kThreads, 0, st>>>(t, p);
    else
      adamw_kernel<false><<<grid, kThreads, 0, st>>>(t, p);
  });
  return cudaGetLastError();
}

cudaError_t launch_adamw_moments_sm100(const uint8_t* m, const uint8_t* m_scale, const uint8_t* v, const uint8_t* v_scale,
                                       long long blocks, void* m_out, void* v_out, int num_sms, cudaStream_t st) {
  adamw_moments_kernel<<<grid_for(blocks, num_sms, 8), kThreads, 0, st>>>(
      m, m_scale, v, v_scale, blocks, static_cast<__nv_bfloat16*>(m_out), static_cast<__nv_bfloat16*>(v_out));
  return cudaGetLastError();
}

}  // namespace dtk
