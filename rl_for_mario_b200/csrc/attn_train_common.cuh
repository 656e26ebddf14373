// Building blocks of the training attention kernels on register fragments:
// swizzled tiles of 16-bit rows brought in with cp.async, ldmatrix, and the
// m16n8k16 product with fp32 accumulators.
#pragma once

#include "dt_common.cuh"
#include "dt_internal.h"
#include "philox.cuh"
#include "prefill_common.cuh"

namespace dtk {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// d += a b for one 16 x 8 x 16 product.
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Rows r0 .. r0 + ROWS of a [*, D] 16-bit matrix (row stride `stride` elements)
// into a swizzled tile.  Rows outside [lo, hi) become zeros and are not read:
// what stands behind the padding never enters a product (0 x NaN would).
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ void load_tile(uint32_t tile, const uint16_t* __restrict__ base, long long stride, int r0,
                                          int lo, int hi, int tid) {
  constexpr int NCH = D / 8;
#pragma unroll
  for (int i = tid; i < ROWS * NCH; i += THREADS) {
    const int r = i / NCH, c = i % NCH, row = r0 + r;
    const bool ok = row >= lo && row < hi;
    cp_async16(tile + swz<D * 2>(r, c), base + (ok ? row * stride + c * 8 : 0), ok);
  }
}

// A fragment (16 rows from r0, 16 columns from 8-column chunk c) of a tile.
template <int D>
__device__ __forceinline__ void frag_a(uint32_t tile, int r0, int c, int lane, uint32_t (&a)[4]) {
  ldsm4(tile + swz<D * 2>(r0 + (lane & 15), c + (lane >> 4)), a);
}
// B fragments of two 8-column blocks, the tile's rows being the columns of B:
// {r0, r1} for rows n0 .. n0 + 8, {r2, r3} for rows n0 + 8 .. n0 + 16.
template <int D>
__device__ __forceinline__ void frag_b(uint32_t tile, int n0, int c, int lane, uint32_t (&b)[4]) {
  ldsm4(tile + swz<D * 2>(n0 + (lane & 7) + ((lane >> 4) << 3), c + ((lane >> 3) & 1)), b);
}
// B fragments of two 8-column blocks, the tile's rows being the rows of B (the
// summed index): {r0, r1} for columns 8 c .., {r2, r3} for columns 8 (c + 1) ..
template <int D>
__device__ __forceinline__ void frag_bt(uint32_t tile, int k0, int c, int lane, uint32_t (&b)[4]) {
  ldsm4_t(tile + swz<D * 2>(k0 + (lane & 15), c + (lane >> 4)), b);
}

}  // namespace dtk
