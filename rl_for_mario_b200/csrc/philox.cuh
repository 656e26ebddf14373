// The dropout generator of the training operators: a counter-based mask that
// is never stored.  Forward and backward evaluate the same function of
// (seed, step, site, element), so a mask costs arithmetic and no memory.
//
// Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011: seven is the fewest rounds of this
// width that pass BigCrush).  key = the 64-bit seed, counter = (block low,
// block high, step, site).  One call gives eight 16-bit words, one for each of
// eight consecutive elements of a row; element (row, col) of a tensor whose
// rows have n columns uses word col % 8 of block row * ceil(n / 8) + col / 8.
// An element stays iff its word >= round(p * 65536), so p is met to 2^-17 and
// survivors are scaled by the exact reciprocal of the rounded rate.
#pragma once

#include <cstdint>

namespace dtk {

struct DropKey {
  uint32_t k0, k1, step, site;
};

// rng points at two 64-bit words, (seed, step); read on the device so that a
// captured graph sees the step of its replay.
__device__ __forceinline__ DropKey drop_key(const long long* __restrict__ rng, uint32_t site) {
  const unsigned long long seed = (unsigned long long)__ldg(rng), step = (unsigned long long)__ldg(rng + 1);
  return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)step, site};
}

__device__ __forceinline__ uint4 philox7(const DropKey& k, unsigned long long block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = k.step, c3 = k.site;
  uint32_t k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    // High and low product words apart: 65 issue slots a call, 84 with 32 x 32 -> 64-bit products (measured).
    const uint32_t ah = __umulhi(c0, 0xD2511F53u), al = c0 * 0xD2511F53u;
    const uint32_t bh = __umulhi(c2, 0xCD9E8D57u), bl = c2 * 0xCD9E8D57u;
    c0 = bh ^ c1 ^ k0;
    c1 = bl;
    c2 = ah ^ c3 ^ k1;
    c3 = al;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Drop flags of a block's eight elements in four words: bit 0 of word i is set when
// element 2 i is dropped, bit 16 when element 2 i + 1 is.  Both halves of a word at
// once: max(w, t) - w is 0 in a half that stays (w >= t), min with 1 makes a flag of
// the rest.  t2 = threshold * 0x10001.
__device__ __forceinline__ uint32_t drop_flags(uint32_t w, uint32_t t2) {
  return __vminu2(__vmaxu2(w, t2) - w, 0x00010001u);
}

// All ones in the halves of four words whose elements stay (word i: elements 2 i and
// 2 i + 1): a pair of 16-bit elements is dropped by one AND.
__device__ __forceinline__ uint4 keep_masks(const DropKey& k, unsigned long long block, uint32_t threshold) {
  const uint4 w = philox7(k, block);
  const uint32_t t2 = threshold * 0x10001u;
  return make_uint4(~(drop_flags(w.x, t2) * 0xffffu), ~(drop_flags(w.y, t2) * 0xffffu),
                    ~(drop_flags(w.z, t2) * 0xffffu), ~(drop_flags(w.w, t2) * 0xffffu));
}

// Bit i set: element i of the block stays.
__device__ __forceinline__ uint32_t keep_bits(const DropKey& k, unsigned long long block, uint32_t threshold) {
  const uint4 w = philox7(k, block);
  const uint32_t t2 = threshold * 0x10001u;
  // Even elements' flags in bits 0, 2, 4, 6, odd ones' in bits 16, 18, 20, 22, then one above the other.
  const uint32_t d = drop_flags(w.x, t2) + drop_flags(w.y, t2) * 4u + drop_flags(w.z, t2) * 16u + drop_flags(w.w, t2) * 64u;
  return ~(d | d >> 15) & 0xffu;
}

// The flags of four blocks (32 elements) in one word, a set bit for a dropped one:
// element e of block b is bit (e & 1) * 16 + 4 b + e / 2 (drop_bit).
__device__ __forceinline__ uint32_t drop_word(const DropKey& k, unsigned long long block, uint32_t threshold) {
  const uint32_t t2 = threshold * 0x10001u;
  uint32_t r = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint4 w = philox7(k, block + b);
    r += (drop_flags(w.x, t2) + drop_flags(w.y, t2) * 2u + drop_flags(w.z, t2) * 4u + drop_flags(w.w, t2) * 8u) << (4 * b);
  }
  return r;
}
__device__ __forceinline__ int drop_place(int element) {  // 0 .. 31
  return (element & 1) * 16 + (element >> 3) * 4 + ((element & 7) >> 1);
}
__device__ __forceinline__ uint32_t drop_bit(int element) { return 1u << drop_place(element); }

// 32 x 32 bits turned over across a warp: bit c of lane b becomes bit b of lane c.
// Five exchanges of half as many bits each time.
__device__ __forceinline__ uint32_t warp_transpose(uint32_t x, int lane) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const uint32_t low = s == 16 ? 0x0000ffffu : s == 8 ? 0x00ff00ffu : s == 4 ? 0x0f0f0f0fu : s == 2 ? 0x33333333u : 0x55555555u;
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, s);
    // The upper lane of a pair takes the other's upper bits into its lower ones, the lower lane the other way.
    x = lane & s ? (x & ~low) | (y >> s & low) : (x & low) | (y << s & ~low);
  }
  return x;
}

}  // namespace dtk
