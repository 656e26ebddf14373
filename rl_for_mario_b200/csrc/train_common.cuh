// Element access shared by the element-wise training kernels: rows of fp32,
// bf16 or fp16 read into and written from fp32 registers, eight columns per
// thread.  VEC: the thread's columns are 8 c .. 8 c + 7 (16-byte accesses, rows
// 16-byte aligned, width a multiple of 8).  Otherwise lane l of warp w owns
// columns 256 w + 32 j + l, j = 0..7 (one element per access, coalesced), which
// takes any width, stride and alignment.
#pragma once

#include <cstdint>

#include "dt_common.cuh"
#include "philox.cuh"

namespace dtk {

// Element codes are the C ABI's: 0 bf16, 1 fp16, 2 fp32.
template <int DT>
struct TrainElem;
template <>
struct TrainElem<0> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to_f(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from_f(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct TrainElem<1> {
  using T = __half;
  static __device__ __forceinline__ float to_f(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from_f(float v) { return __float2half_rn(v); }
};
template <>
struct TrainElem<2> {
  using T = float;
  static __device__ __forceinline__ float to_f(T v) { return v; }
  static __device__ __forceinline__ T from_f(float v) { return v; }
};

// Eight columns of a row; `w` is the warp's index within the row, n its width.
// Columns at or past n read as 0 and are not written.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const typename TrainElem<DT>::T* __restrict__ row, int w, int lane, int n,
                                      float (&v)[8]) {
  if constexpr (VEC) {
    const int c = (w * 32 + lane) * 8;
    if (c < n) {
      if constexpr (DT == 2) {
        const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 u = *reinterpret_cast<const uint4*>(row + c);
        const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Elem<DT == 0>::to_f2(q[i]);
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = w * 256 + j * 32 + lane;
      v[j] = c < n ? TrainElem<DT>::to_f(row[c]) : 0.f;
    }
  }
}

// The same eight columns as they stand in memory: what a thread holds of a row that
// it works on later (half the registers of fp32 for 16-bit rows of vectors).
template <int DT, bool VEC>
struct Raw8 {
  using T = typename TrainElem<DT>::T;
  float v[8];
  __device__ __forceinline__ void load(const T* __restrict__ row, int w, int lane, int n) {
    load8<DT, VEC>(row, w, lane, n, v);
  }
  __device__ __forceinline__ void get(float (&o)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = v[i];
  }
};
template <int DT>
struct Raw8Half {
  using T = typename TrainElem<DT>::T;
  uint4 u;
  __device__ __forceinline__ void load(const T* __restrict__ row, int w, int lane, int n) {
    const int c = (w * 32 + lane) * 8;
    u = c < n ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&o)[8]) const {
    const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<DT == 0>::to_f2(q[i]);
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Raw8<0, true> : Raw8Half<0> {};
template <>
struct Raw8<1, true> : Raw8Half<1> {};

template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename TrainElem<DT>::T* __restrict__ row, int w, int lane, int n,
                                       const float (&v)[8]) {
  if constexpr (VEC) {
    const int c = (w * 32 + lane) * 8;
    if (c < n) {
      if constexpr (DT == 2) {
        *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        using E = Elem<DT == 0>;
        *reinterpret_cast<uint4*>(row + c) = make_uint4(E::from_f2(v[0], v[1]), E::from_f2(v[2], v[3]),
                                                        E::from_f2(v[4], v[5]), E::from_f2(v[6], v[7]));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = w * 256 + j * 32 + lane;
      if (c < n) row[c] = TrainElem<DT>::from_f(v[j]);
    }
  }
}

// Eight columns as packed pairs (one instruction for two of them: the kernels are
// as near to the issue rate as to HBM).
struct F8 {
  float2 p[4];
  template <int DT, bool VEC>
  __device__ __forceinline__ void load(const typename TrainElem<DT>::T* row, int w, int lane, int n) {
    load8<DT, VEC>(row, w, lane, n, as());
  }
  __device__ __forceinline__ float (&as())[8] { return *reinterpret_cast<float(*)[8]>(p); }
  __device__ __forceinline__ void set(float v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = make_float2(v, v);
  }
  // Clears what the mask bits drop (bit i: element i stays).
  __device__ __forceinline__ void keep(uint32_t m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i].x = (m >> (2 * i)) & 1u ? p[i].x : 0.f;
      p[i].y = (m >> (2 * i + 1)) & 1u ? p[i].y : 0.f;
    }
  }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float both_sum(float2 v) { return v.x + v.y; }

// Bit i set: the thread's element i stays.  Every lane computes the block of
// columns 8 (32 w + lane) ..; without VEC the bits then move to the lanes that
// own the columns (element j of lane l is bit l % 8 of lane 4 j + l / 8).
template <bool VEC>
__device__ __forceinline__ uint32_t keep8(const DropKey& key, unsigned long long row_block, int w, int lane,
                                          uint32_t threshold) {
  const uint32_t m = keep_bits(key, row_block + (unsigned)(w * 32 + lane), threshold);
  if constexpr (VEC) {
    return m;
  } else {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      r |= ((__shfl_sync(0xffffffffu, m, j * 4 + (lane >> 3)) >> (lane & 7)) & 1u) << j;
    return r;
  }
}

}  // namespace dtk
