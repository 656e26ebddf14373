// The end of a training step over all of a model's tensors at once: the norm of the
// gradient and the AdamW update (Loshchilov, Hutter, ICLR 2019), clipped by it.
//
//   c = min(1, max_norm / (norm + 1e-6)),  g' = c g
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)      t the step, from 1
//
// Tensors are cut into blocks of 256 elements, a warp's work; a tensor starts a new block, so
// the averages of tensor i lie from element 256 (blocks before it) on in flat arrays of whole
// blocks.  Pointers and sizes travel as kernel arguments (up to 768 tensors a launch): there
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
// Bound by HBM: an element of a bf16 weight costs 22 bytes with 32-bit averages, 10 with 8-bit ones, 28 with 32-bit
// averages and fp32 weights beside it.  81.3 M weights in 125 tensors, inputs cold: 32-bit averages 293 us in bf16
// (6.1 TB/s), 385 in fp32 (28 bytes, 5.9), 387 in bf16 with fp32 weights (5.9); 8-bit ones 215 us with fp32 weights
// beside bf16 ones (16 bytes, 6.0), 213 in fp32 (6.1), 174 in bf16 alone (4.7 TB/s): there the codes' work, 375 warp
// instructions a block of 256 elements, takes 63 % of the issue slots and 50 % of the ALU pipe with 18 warps on an SM,
// and a warp waits for its loads in 2.1 of the 7 cycles between two of its instructions.
#include <cstring>
#include <type_traits>

#include "dt_common.cuh"
#include "dt_internal.h"
#include "philox.cuh"
#include "train_common.cuh"

namespace dtk {

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
// Blocks on an SM.  Norm, 81.3 M bf16 numbers: 41 us with 8, 45 with 6, 45 with 12 (spills).  Step: what leaves the loads of
// two blocks their registers; 32-bit averages, bf16 weights: 292 us with 4, 300 with 6; 8-bit ones 175 with 5 (12 bytes
// of spills), 184 to 187 with 6 (more), 192 to 197 with 4.
constexpr int kNormResident = 8;
template <bool BITS8, bool MASTER = false>
constexpr int kStepResident = BITS8 && !MASTER ? 5 : 4;
constexpr int kNormUnit = 1024;      // elements of a warp's turn in the norm
constexpr int kPair = 512;           // of two blocks, whose loads are in flight together in the step
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

// Eight elements as they stand in memory (one 16-byte word of 16-bit ones, two of fp32), on their way while
// others are worked on.
struct Raw8Any {
  uint4 u[2];
};
__device__ __forceinline__ Raw8Any get_raw(int code, const void* base, long long at, long long n, bool vec) {
  Raw8Any r;
  r.u[0] = r.u[1] = make_uint4(0u, 0u, 0u, 0u);
  if (vec && at + 8 <= n) {
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * (code == 2 ? 4 : 2));
    r.u[0] = x[0];
    if (code == 2) r.u[1] = x[1];
  } else if (at < n) {  // an address off the boundary, or the tensor's end: elements past it read as 0
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
    if (code == 2) {
      const uint32_t* x = static_cast<const uint32_t*>(base) + at;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < n) w[i] = x[i];
    } else {
      const uint16_t* x = static_cast<const uint16_t*>(base) + at;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < n) w[i >> 1] |= (uint32_t)x[i] << (16 * (i & 1));
    }
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.u[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return r;
}
__device__ __forceinline__ void unpack(int code, const Raw8Any& r, F8& v) {
  const uint32_t w[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v.p[i] = code == 2   ? make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]))
             : code == 1 ? Elem<false>::to_f2(w[i])
                         : Elem<true>::to_f2(w[i]);
}
// The elements rounded to their type; those past the tensor's end are not written.
__device__ __forceinline__ void put8(int code, void* base, long long at, long long n, bool vec, const F8& v) {
  if (code == 2) {
    float* x = static_cast<float*>(base) + at;
    if (vec && at + 8 <= n) {
      *reinterpret_cast<float4*>(x) = make_float4(v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y);
      *reinterpret_cast<float4*>(x + 4) = make_float4(v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < n) x[i] = i & 1 ? v.p[i >> 1].y : v.p[i >> 1].x;
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = code == 1 ? Elem<false>::from_f2(v.p[i].x, v.p[i].y) : Elem<true>::from_f2(v.p[i].x, v.p[i].y);
    uint16_t* x = static_cast<uint16_t*>(base) + at;
    if (vec && at + 8 <= n) {
      *reinterpret_cast<uint4*>(x) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < n) x[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
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
// Two squares are added in fp32 (of 16-bit numbers they are exact), the sums of pairs in fp64: the rounded
// norm is then the exact one's in all but one case of some thousands, and with it the clipped averages to
// the last bit (sums of 32 squares in fp32: one in a hundred).  Squares of numbers beyond 2^63 overflow in fp32,
// those of numbers below 2^-63 lose their bits: a lane that meets such takes its 32 again in fp64.
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
    const int code = s.kind & 3;
    const long long first = (long long)(u - (t ? ends[t - 1] : 0u)) * kNormUnit + lane * 8;
    const bool vec = aligned16(s.g);
    constexpr int TURNS = kNormUnit / 256;
    Raw8Any raw[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) raw[i] = get_raw(code, s.g, first + i * 256, s.n, vec);
    double d[2] = {0.0, 0.0};
    auto squares = [&](auto code) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        F8 v;
        unpack(code.value, raw[i], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j & 1] += (double)both_sum(fmul2(v.p[j], v.p[j]));
      }
    };
    if (code == 0) squares(std::integral_constant<int, 0>{});
    else if (code == 1) squares(std::integral_constant<int, 1>{});
    else squares(std::integral_constant<int, 2>{});
    const double all = d[0] + d[1];
    if (all >= 1e-28 && all <= 1e38) {
      sum += all;
    } else {
#pragma unroll 1
      for (int i = 0; i < TURNS; ++i) {
        F8 v;
        unpack(code, get_raw(code, s.g, first + i * 256, s.n, vec), v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum += (double)v.p[j].x * (double)v.p[j].x + (double)v.p[j].y * (double)v.p[j].y;
      }
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

// Eight codes of the first (second) average as fp32, times f.
__device__ __forceinline__ void decode_first(uint2 codes, float f, F8& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)((i < 2 ? codes.x : codes.y) >> (16 * (i & 1)))));
    v.p[i] = fmul2(__half22float2(*reinterpret_cast<__half2*>(&h)), both(f));
  }
}
__device__ __forceinline__ void decode_second(uint2 codes, float f, F8& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // Two codes, each 7 bits up in a half of its own.
    uint32_t h = __byte_perm(i < 2 ? codes.x : codes.y, 0, i & 1 ? 0x4342 : 0x4140) << 7;
    v.p[i] = fmul2(__half22float2(*reinterpret_cast<__half2*>(&h)), both(f));
  }
}

// The largest of three numbers, or NaN when one of them is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// y >= 0, scaled into the codes' range (below 2^(TOP + 1)), rounded up or down at random to three bits behind
// the leading one: the code comes out as the top byte.  An fp32 number shifted up by four bits has its
// exponent's lower five bits and its three leading ones there, and 20 more below; adding the word at the
// top of these carries into the code in the part's proportion.  The exponent's bias changes by the byte that
// `word` has above the 16 random bits.  Numbers below 2^(1 - BIAS) have equal steps of 2^(-2 - BIAS): 2^(1 - BIAS) is
// added first, after which they stand in the binade with that spacing, eight codes up (rounded to zero:
// what falls off lies below the random bits).  The comparison's result as the number 1 or 0 does both on the
// FMA pipe: the ALU, at half its rate, is what the 8-bit step runs into.
template <int BIAS>
__device__ __forceinline__ uint32_t encode(float y, uint32_t word, uint32_t select) {
  constexpr float low = 1.f / (1 << (BIAS - 1));
  constexpr uint32_t back = (uint32_t)(-((127 - BIAS) << 3)) & 0xffu;
  // The bits of 1.0f times this are -8 in the top byte: 127 * 2^23 * 16 mod 2^32 = -2^27.
  constexpr uint32_t eight = 16u;
  static_assert(0x3f800000u * eight == (uint32_t)(-8) << 24, "");
  float small;
  asm("set.lt.f32.f32 %0, %1, %2;" : "=f"(small) : "f"(y), "f"(low));
  const float z = __fmaf_rz(small, low, y);
  return __float_as_uint(z) * 16u + (__float_as_uint(small) * eight + __byte_perm(word, back, select));
}

// Stores a lane's eight values of a block; returns the block's scale.  Random words: the two halves of each word,
// the bytes of a half turned over for the signed average.
template <int BIAS, int TOP, bool SIGNED>
__device__ __forceinline__ int put_codes(uint8_t* codes, const F8& x, const uint4& words) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max_nan(most, fabsf(x.p[i].x), fabsf(x.p[i].y));
  const int e = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23), kMinScale);
  const float f = scale_of(254 + TOP - min(e, 254));
  const uint32_t w[4] = {words.x, words.y, words.z, words.w};
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = fmul2(x.p[i], both(f));
    // Bytes: 0, the half's two, the bias.
    c[2 * i] = encode<BIAS>(SIGNED ? fabsf(y.x) : y.x, w[i], SIGNED ? 0x4015 : 0x4105);
    c[2 * i + 1] = encode<BIAS>(SIGNED ? fabsf(y.y) : y.y, w[i], SIGNED ? 0x4235 : 0x4325);
    if constexpr (SIGNED) {
      c[2 * i] = (c[2 * i] & 0x7fffffffu) | (__float_as_uint(y.x) & 0x80000000u);
      c[2 * i + 1] = (c[2 * i + 1] & 0x7fffffffu) | (__float_as_uint(y.y) & 0x80000000u);
    }
  }
  uint32_t four[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    four[k] = __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0073), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0073), 0x5410);
    if constexpr (!SIGNED)
      if ((four[k] - 0x01010101u) & ~four[k] & 0x80808080u)  // a zero among them: a step for what is above zero
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = j & 1 ? x.p[2 * k + (j >> 1)].y : x.p[2 * k + (j >> 1)].x;
          if (v > 0.f && !(four[k] >> (8 * j) & 0xffu)) four[k] |= 1u << (8 * j);
        }
  }
  *reinterpret_cast<uint2*>(codes) = make_uint2(four[0], four[1]);
  return e;
}

// ---------------------------------------------------------------- step
struct GroupNow {
  float rate, root, decay, b1, c1, b2, c2, eps;
};

// Each off by an ulp or so; the weights' own rounding is larger than what that does to a step.  FLUSH: numbers below the
// normal ones, whose root is below 2^-63, count as zero (flushes_roots says where that is nothing beside eps): one
// instruction instead of five.
template <bool FLUSH>
__device__ __forceinline__ float fast_sqrt(float x) {
  float r;
  if constexpr (FLUSH)
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  else
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_inverse(float x) {  // of normal numbers (eps is one)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What a lane holds of a block of 256 elements.
template <bool BITS8>
struct BlockLoad {
  Raw8Any g, w;
  uint4 m[BITS8 ? 1 : 2], v[BITS8 ? 1 : 2];  // 8 bits: codes in x, y
};

// The scales of a unit's blocks: lane i holds those of block i, so that a unit reads and writes them in one
// access each.  (Byte by byte with each block, 81 M bf16 weights took 205 us: loads and stores of neighbouring
// bytes by many warps get in each other's way.)
struct Scales {
  int m, v;
};

// A block's place: of the lane's first element in its tensor and in the flat arrays.
struct BlockPlace {
  long long at, block;
  __device__ __forceinline__ long long mine(int lane) const { return block * 256 + lane * 8; }
};

// CODE: the tensor's element code; VEC: the block is whole and stands on 16-byte boundaries.
template <bool BITS8, bool MASTER, int CODE, bool VEC>
__device__ __forceinline__ BlockLoad<BITS8> load_block(const AdamWParams& p, const TensorSlot& s, const BlockPlace& q, int lane) {
  BlockLoad<BITS8> r;
  const long long mine = q.mine(lane), end = VEC ? q.at + 8 : s.n;
  r.g = get_raw(CODE, s.g, q.at, end, VEC || aligned16(s.g));
  if constexpr (MASTER && CODE != 2)
    r.w = get_raw(2, p.master, mine, mine + 8, true);
  else
    r.w = get_raw(CODE, s.p, q.at, end, VEC || aligned16(s.p));
  if constexpr (BITS8) {
    const uint2 m = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.m) + mine);
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.v) + mine);
    r.m[0] = make_uint4(m.x, m.y, 0u, 0u);
    r.v[0] = make_uint4(v.x, v.y, 0u, 0u);
  } else {
    const Raw8Any m = get_raw(2, p.m, mine, mine + 8, true), v = get_raw(2, p.v, mine, mine + 8, true);
    r.m[0] = m.u[0], r.m[1] = m.u[1], r.v[0] = v.u[0], r.v[1] = v.u[1];
  }
  return r;
}

template <bool BITS8, bool MASTER, bool FLUSH, int CODE, bool VEC>
__device__ __forceinline__ void step_block(const AdamWParams& p, const TensorSlot& s, const BlockPlace& place, int number,
                                           Scales& scales, const BlockLoad<BITS8>& r, const GroupNow& q, float clip,
                                           const DropKey& key, int lane) {
  const long long mine = place.mine(lane);
  F8 w, h, m, v;
  unpack(CODE, r.g, h);
  unpack(MASTER ? 2 : CODE, r.w, w);
  // The averages times b1 and b2: in 8 bits scale and factor in one, which rounds the same.
  if constexpr (BITS8) {
    decode_first(make_uint2(r.m[0].x, r.m[0].y), decode_scale<7>(__shfl_sync(0xffffffffu, scales.m, number)) * q.b1, m);
    decode_second(make_uint2(r.v[0].x, r.v[0].y), decode_scale<14>(__shfl_sync(0xffffffffu, scales.v, number)) * q.b2, v);
  } else {
    unpack(2, Raw8Any{r.m[0], r.m[1]}, m);
    unpack(2, Raw8Any{r.v[0], r.v[1]}, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) m.p[i] = fmul2(m.p[i], both(q.b1)), v.p[i] = fmul2(v.p[i], both(q.b2));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // Each product and sum of the averages is rounded by itself, so that what is stored is one well-defined number.
    // (The sums are written as a product with one plus the other: a packed product and the sum behind it would be
    // contracted for all their .rn, and `one` is an argument that the compiler does not know.)
    h.p[i] = fmul2(h.p[i], both(clip));
    m.p[i] = ffma2(fmul2(h.p[i], both(q.c1)), both(p.one), m.p[i]);
    v.p[i] = ffma2(fmul2(fmul2(h.p[i], h.p[i]), both(q.c2)), both(p.one), v.p[i]);
    const float2 d = make_float2(fast_inverse(fmaf(fast_sqrt<FLUSH>(v.p[i].x), q.root, q.eps)),
                                 fast_inverse(fmaf(fast_sqrt<FLUSH>(v.p[i].y), q.root, q.eps)));
    w.p[i] = ffma2(fmul2(m.p[i], both(-q.rate)), d, fmul2(w.p[i], both(q.decay)));
  }
  if constexpr (MASTER && CODE != 2) put8(2, p.master, mine, mine + 8, true, w);
  put8(CODE, s.p, place.at, VEC ? place.at + 8 : s.n, VEC || aligned16(s.p), w);
  if constexpr (BITS8) {
    const uint4 u = philox7(key, (unsigned long long)place.block * 32 + lane);
    const int em = put_codes<7, 7, true>(static_cast<uint8_t*>(p.m) + mine, m, u);
    const int ev = put_codes<15, 14, false>(static_cast<uint8_t*>(p.v) + mine, v, u);
    if (lane == number) scales = Scales{em, ev};
  } else {
    put8(2, p.m, mine, mine + 8, true, m);
    put8(2, p.v, mine, mine + 8, true, v);
  }
}

// A warp's unit of work: pairs of blocks, or what the tensor has left of them.
template <bool BITS8, bool MASTER, bool FLUSH, int CODE>
__device__ __forceinline__ void step_unit(const AdamWParams& p, const TensorSlot& s, uint32_t unit, float clip,
                                          const GroupNow* groups, const DropKey& key, int lane) {
  const GroupNow q = groups[s.kind >> 8];
  const bool vec = aligned16(s.p) && aligned16(s.g);
  const int pairs = BITS8 ? p.pairs : 1;
  long long first = (long long)unit * pairs * kPair;
  BlockPlace a{first + lane * 8, p.first + s.first + first / 256};
  const long long block = a.block;
  const bool scaled = BITS8 && lane < 2 * pairs && first + lane * 256 < s.n;  // of the lane's block
  Scales scales{0, 0};
  if (scaled) scales = Scales{p.m_scale[block + lane], p.v_scale[block + lane]};
#pragma unroll 1
  for (int k = 0; k < pairs && first < s.n; ++k, first += kPair) {
    const BlockPlace b{a.at + 256, a.block + 1};
    if (vec && first + kPair <= s.n) {
      const auto x = load_block<BITS8, MASTER, CODE, true>(p, s, a, lane), y = load_block<BITS8, MASTER, CODE, true>(p, s, b, lane);
      step_block<BITS8, MASTER, FLUSH, CODE, true>(p, s, a, 2 * k, scales, x, q, clip, key, lane);
      step_block<BITS8, MASTER, FLUSH, CODE, true>(p, s, b, 2 * k + 1, scales, y, q, clip, key, lane);
    } else {
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const BlockPlace& c = i ? b : a;
        if (first + i * 256 < s.n)
          step_block<BITS8, MASTER, FLUSH, CODE, false>(p, s, c, 2 * k + i, scales,
                                                        load_block<BITS8, MASTER, CODE, false>(p, s, c, lane), q, clip, key,
                                                        lane);
      }
    }
    a.at += kPair;
    a.block += 2;
  }
  if (scaled) p.m_scale[block + lane] = (uint8_t)scales.m, p.v_scale[block + lane] = (uint8_t)scales.v;
}

// x^n by squaring.
__device__ __forceinline__ double power(double x, unsigned long long n) {
  double r = 1.0;
  for (; n; n >>= 1, x *= x)
    if (n & 1) r *= x;
  return r;
}

template <bool BITS8, bool MASTER, bool FLUSH, int N>
__global__ void __launch_bounds__(kThreads, kStepResident<BITS8, MASTER>) adamw_kernel(const __grid_constant__ TensorTable<N> table,
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
    for (uint32_t u = blockIdx.x * kWarps + (threadIdx.x >> 5); u < p.units; u += gridDim.x * kWarps) {
      const int t = find_slot(ends, p.count, u, lane);
      const TensorSlot& s = table.slot[t];
      if (!s.g) continue;
      const uint32_t unit = u - (t ? ends[t - 1] : 0u);
      const int code = s.kind & 3;
      if (code == 0) step_unit<BITS8, MASTER, FLUSH, 0>(p, s, unit, clip, groups, key, lane);
      else if (code == 1) step_unit<BITS8, MASTER, FLUSH, 1>(p, s, unit, clip, groups, key, lane);
      else step_unit<BITS8, MASTER, FLUSH, 2>(p, s, unit, clip, groups, key, lane);
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
    F8 x, y;
    decode_first(*reinterpret_cast<const uint2*>(m + at), decode_scale<7>(m_scale[b]), x);
    decode_second(*reinterpret_cast<const uint2*>(v + at), decode_scale<14>(v_scale[b]), y);
    put8(0, m_out, at, at + 8, true, x);
    put8(0, v_out, at, at + 8, true, y);
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

// (What four warps take in four turns is one block's, which needs no second launch for the sum.)
int grad_norm_grid(long long units, int num_sms) {
  return units <= 4 * kWarps ? 1 : (int)grid_for(units, num_sms, kNormResident);
}
long long grad_norm_unit() { return kNormUnit; }
int adamw_pairs(long long blocks, int state_bits, int num_sms) {
  // 8 bits: units of four pairs have their scales in one access, units of one leave more warps something to do.  bf16
  // weights in eight tensors, one pair against four: 1 M 11.3 us and 15.4, 5 M 21 and 21.5, 10 M 31.8 and 29.7, 18 M
  // 52 and 46, 80 M 206 and 171 (two pairs 183, eight 183, sixteen 204); so four from one and a half for each warp on.
  // 32 bits: one (two pairs 2 to 4 % slower, four 4 %: neighbouring warps then read further apart).
  const long long warps = (long long)num_sms * kWarps * kStepResident<true>;
  return state_bits == 8 && blocks >= 12 * warps ? 4 : 1;
}

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

namespace {

// 8 bits: whether roots of averages below the normal numbers may be taken as zero.  A root is below 2^-63 there and counts
// at most 1 / sqrt(1 - b2) times; eps, which it is added to, has to be 2^25 times that in every group (1.2e-10 with b2 = 0.999).
// 81 M bf16 weights: 174 us with it, 182 without, with fp32 weights beside them 215 and 219, fp32 weights 213 both ways.
// (32-bit averages, bound by HBM, take every root.)
bool flushes_roots(const AdamWParams& p) {
  if (!p.m_scale) return false;
  for (int i = 0; i < p.ngroups; ++i)
    if (!(p.group[i].eps * sqrt(1.0 - p.group[i].b2) >= 0x1p-38)) return false;
  return true;
}

template <bool BITS8, bool MASTER, bool FLUSH>
cudaError_t launch_adamw(const TensorSlot* slots, const AdamWParams& p, int num_sms, cudaStream_t st) {
  const unsigned grid = grid_for(p.units, num_sms, kStepResident<BITS8, MASTER>);
  with_tables(slots, p.count, [&](const auto& t) {
    adamw_kernel<BITS8, MASTER, FLUSH><<<grid, kThreads, 0, st>>>(t, p);
  });
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adamw_sm100(const TensorSlot* slots, const AdamWParams& p, int num_sms, cudaStream_t st) {
  if (!p.m_scale)
    return p.master ? launch_adamw<false, true, false>(slots, p, num_sms, st)
                    : launch_adamw<false, false, false>(slots, p, num_sms, st);
  if (flushes_roots(p))
    return p.master ? launch_adamw<true, true, true>(slots, p, num_sms, st)
                    : launch_adamw<true, false, true>(slots, p, num_sms, st);
  return p.master ? launch_adamw<true, true, false>(slots, p, num_sms, st)
                  : launch_adamw<true, false, false>(slots, p, num_sms, st);
}

cudaError_t launch_adamw_moments_sm100(const uint8_t* m, const uint8_t* m_scale, const uint8_t* v, const uint8_t* v_scale,
                                       long long blocks, void* m_out, void* v_out, int num_sms, cudaStream_t st) {
  adamw_moments_kernel<<<grid_for(blocks, num_sms, 8), kThreads, 0, st>>>(
      m, m_scale, v, v_scale, blocks, static_cast<__nv_bfloat16*>(m_out), static_cast<__nv_bfloat16*>(v_out));
  return cudaGetLastError();
}

}  // namespace dtk
