// Causal grouped-query attention for training, with its gradient.
//
// For a query row q >= pad of head h (KV head g = h / R) and keys j in pad..q:
//   s_j = scale q . k_j,   P_j = exp(s_j) / sum exp,   O = sum_j m_j P_j v_j / (1 - p)
// with m the dropout mask (philox.cuh).  Rows q < pad see no key: O = 0, no
// gradient.  Backward, with m' = m / (1 - p):
//   dV_j = sum_q m' P dO,   dP_j = m' dO . v_j,   delta = sum_j P_j dP_j = O . dO
//   dS_j = P_j (dP_j - delta),   dq = scale sum_j dS_j k_j,   dk_j = scale sum_q dS_j q
// The forward pass keeps log2 sum exp2 of each row (base-2 logarithm of the
// softmax's denominator), so the backward passes form P again from one product.
//
// Two backward kernels: one walks the keys of 64 query rows (delta and dq), one
// walks the query rows of all R heads behind 64 keys (dk and dv).  Each sum has
// one owner, so there are no atomics and every run gives the same bits; the
// price is that S and dP are formed twice.
//
// Rounding: P and dS enter the second products in the inputs' 16-bit type, as
// the tensor cores take both operands in one type; sums, softmax statistics
// and delta are fp32.  A row with a single key has a constant softmax: its dS
// is set to exactly zero.  Where a row's keys lie in one tile delta is the sum
// over the unrounded P dP; beyond, it is O . dO with the stored O.
#include "attn_train_common.cuh"

namespace dtk {

namespace {

constexpr int kT = 64;        // query rows and keys of a tile
constexpr int kThreads = 128;


// Keep bits of a warp's 16 query rows x 64 keys: lane l holds 32 bits, blocks
// 4 (l / 16) .. + 4 of row l % 16.
__device__ __forceinline__ uint32_t keep_rows(const DropKey& key, unsigned long long row_block0, unsigned per_row,
                                              int lane, uint32_t threshold) {
  const unsigned long long b = row_block0 + (unsigned long long)(lane & 15) * per_row + (lane >> 4) * 4;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= keep_bits(key, b + i, threshold) << (8 * i);
  return m;
}

template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kThreads) attn_train_fwd_kernel(const AttnTrainParams p, int ntiles) {
  constexpr int TB = kT * D * 2;
  __shared__ __align__(1024) uint8_t smem[5 * TB];
  const uint32_t sq = smem_u32(smem), sk = sq + TB, sv = sq + 3 * TB;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int qt = ntiles - 1 - (int)(blockIdx.x % (unsigned)ntiles);
  const unsigned bh = blockIdx.x / (unsigned)ntiles;
  const int b = (int)(bh / (unsigned)p.Hq), h = (int)(bh % (unsigned)p.Hq), g = h / p.R;
  const int S = p.S, q0 = qt * kT;
  const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), S) : 0;
  const int q_end = min(S, q0 + kT);
  uint16_t* o = static_cast<uint16_t*>(p.o) + b * p.o_sb + h * p.o_sh;
  float* lse = p.lse + ((long long)b * p.Hq + h) * S;
  using E = Elem<BF16>;

  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float c2 = p.scale * 1.4426950408889634f;

  if (q_end > pad) {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb + h * p.q_sh;
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + b * p.k_sb + g * p.k_sh;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.v_sb + g * p.v_sh;
    DropKey key{};
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    unsigned long long blk = 0;
    if constexpr (DROP) {
      key = drop_key(p.rng, p.site);
      blk = ((unsigned long long)bh * (unsigned)S + (unsigned)(q0 + warp * 16)) * per_row;
    }
    const int kt0 = pad / kT;
    load_tile<D, kT, kThreads>(sq, q, p.q_ss, q0, pad, S, tid);
    load_tile<D, kT, kThreads>(sk, k, p.k_ss, kt0 * kT, pad, S, tid);
    load_tile<D, kT, kThreads>(sv, v, p.v_ss, kt0 * kT, pad, S, tid);
    cp_async_commit();
    uint32_t qa[D / 16][4];
    for (int kt = kt0; kt <= qt; ++kt) {
      const int buf = (kt - kt0) & 1;
      cp_async_wait<0>();
      __syncthreads();
      if (kt < qt) {
        load_tile<D, kT, kThreads>(sk + (buf ^ 1) * TB, k, p.k_ss, (kt + 1) * kT, pad, S, tid);
        load_tile<D, kT, kThreads>(sv + (buf ^ 1) * TB, v, p.v_ss, (kt + 1) * kT, pad, S, tid);
        cp_async_commit();
      }
      if (kt == kt0)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) frag_a<D>(sq, warp * 16, 2 * i, lane, qa[i]);
      float s[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t bb[4];
          frag_b<D>(sk + buf * TB, 16 * j, 2 * i, lane, bb);
          mma16816<BF16>(s[2 * j], qa[i], bb[0], bb[1]);
          mma16816<BF16>(s[2 * j + 1], qa[i], bb[2], bb[3]);
        }
      if (kt == qt || kt * kT < pad) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kk = kt * kT + 8 * j + 2 * t4 + (e & 1), qq = q0 + warp * 16 + g8 + (e >> 1) * 8;
            if (kk > qq || kk < pad) s[j][e] = -INFINITY;
          }
      }
      float mu[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = m[r];
#pragma unroll
        for (int j = 0; j < 8; ++j) x = fmaxf(x, fmaxf(s[j][2 * r], s[j][2 * r + 1]) * c2);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mu[r] = x == -INFINITY ? 0.f : x;
        const float f = ex2_approx(m[r] - mu[r]);
        m[r] = x;
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          acc[i][2 * r] *= f;
          acc[i][2 * r + 1] *= f;
        }
      }
      uint32_t keep = 0xffffffffu;
      if constexpr (DROP) keep = keep_rows(key, blk + (unsigned)kt * (kT / 8), per_row, lane, p.threshold);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x0 = ex2_approx(fmaf(s[j][2 * r], c2, -mu[r])), x1 = ex2_approx(fmaf(s[j][2 * r + 1], c2, -mu[r]));
          l[r] += x0 + x1;
          if constexpr (DROP) {
            const uint32_t bits = __shfl_sync(0xffffffffu, keep, g8 + 8 * r + (j >> 2) * 16) >> ((j & 3) * 8 + 2 * t4);
            s[j][2 * r] = bits & 1u ? x0 : 0.f;
            s[j][2 * r + 1] = bits & 2u ? x1 : 0.f;
          } else {
            s[j][2 * r] = x0;
            s[j][2 * r + 1] = x1;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a[4] = {E::from_f2(s[2 * j][0], s[2 * j][1]), E::from_f2(s[2 * j][2], s[2 * j][3]),
                               E::from_f2(s[2 * j + 1][0], s[2 * j + 1][1]),
                               E::from_f2(s[2 * j + 1][2], s[2 * j + 1][3])};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t bb[4];
          frag_bt<D>(sv + buf * TB, 16 * j, 2 * i, lane, bb);
          mma16816<BF16>(acc[2 * i], a, bb[0], bb[1]);
          mma16816<BF16>(acc[2 * i + 1], a, bb[2], bb[3]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = q0 + warp * 16 + g8 + 8 * r;
    float sum = l[r];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (row >= S) continue;
    const float inv = sum > 0.f ? p.inv_keep / sum : 0.f;
    if (t4 == 0) lse[row] = sum > 0.f ? m[r] + log2f(sum) : INFINITY;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<uint32_t*>(o + row * p.o_ss + 8 * i + 2 * t4) =
          E::from_f2(acc[i][2 * r] * inv, acc[i][2 * r + 1] * inv);
  }
}

// delta and dq of 64 query rows of one head.
template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kThreads) attn_train_dq_kernel(const AttnTrainParams p, int ntiles) {
  constexpr int TB = kT * D * 2;
  __shared__ __align__(1024) uint8_t smem[5 * TB];
  __shared__ float sdelta[kT];
  const uint32_t sq = smem_u32(smem), sk = sq + TB, sv = sq + 3 * TB;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int qt = ntiles - 1 - (int)(blockIdx.x % (unsigned)ntiles);
  const unsigned bh = blockIdx.x / (unsigned)ntiles;
  const int b = (int)(bh / (unsigned)p.Hq), h = (int)(bh % (unsigned)p.Hq), g = h / p.R;
  const int S = p.S, q0 = qt * kT;
  const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), S) : 0;
  const int q_end = min(S, q0 + kT);
  uint16_t* dq = static_cast<uint16_t*>(p.dq) + b * p.dq_sb + h * p.dq_sh;
  using E = Elem<BF16>;

  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

  if (q_end > pad) {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb + h * p.q_sh;
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + b * p.k_sb + g * p.k_sh;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.v_sb + g * p.v_sh;
    const uint16_t* dout = static_cast<const uint16_t*>(p.dout) + b * p.do_sb + h * p.do_sh;
    const float c2 = p.scale * 1.4426950408889634f;
    const int kt0 = pad / kT;
    const bool one_tile = kt0 == qt;
    // Q and dO pass through the second K / V buffers into registers.
    load_tile<D, kT, kThreads>(sk + TB, q, p.q_ss, q0, pad, S, tid);
    load_tile<D, kT, kThreads>(sv + TB, dout, p.do_ss, q0, pad, S, tid);
    load_tile<D, kT, kThreads>(sk, k, p.k_ss, kt0 * kT, pad, S, tid);
    load_tile<D, kT, kThreads>(sv, v, p.v_ss, kt0 * kT, pad, S, tid);
    cp_async_commit();
    const long long row0 = (long long)bh * S;
    if (!one_tile) {
      // delta = O . dO, two threads a row.
      const uint16_t* o = static_cast<const uint16_t*>(p.o) + b * p.o_sb + h * p.o_sh;
      const int r = tid >> 1, row = q0 + r;
      float d = 0.f;
      if (row >= pad && row < S) {
        const uint4* po = reinterpret_cast<const uint4*>(o + row * p.o_ss + (tid & 1) * (D / 2));
        const uint4* pd = reinterpret_cast<const uint4*>(dout + row * p.do_ss + (tid & 1) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint4 a = __ldg(po + i), c = __ldg(pd + i);
          const uint32_t au[4] = {a.x, a.y, a.z, a.w}, cu[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = E::to_f2(au[e]), y = E::to_f2(cu[e]);
            d = fmaf(x.x, y.x, fmaf(x.y, y.y, d));
          }
        }
      }
      d += __shfl_xor_sync(0xffffffffu, d, 1);
      if (!(tid & 1)) {
        sdelta[r] = d;
        if (row < S) p.delta[row0 + row] = d;
      }
    }
    DropKey key{};
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    unsigned long long blk = 0;
    if constexpr (DROP) {
      key = drop_key(p.rng, p.site);
      blk = ((unsigned long long)bh * (unsigned)S + (unsigned)(q0 + warp * 16)) * per_row;
    }
    float ls[2], delta[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // A row with one key (row == pad) has no gradient: P is taken as 0.
      const int row = q0 + warp * 16 + g8 + 8 * r;
      ls[r] = row < S && row != pad ? __ldg(p.lse + row0 + row) : INFINITY;
    }
    cp_async_wait<0>();
    __syncthreads();
    uint32_t qa[D / 16][4], da[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      frag_a<D>(sk + TB, warp * 16, 2 * i, lane, qa[i]);
      frag_a<D>(sv + TB, warp * 16, 2 * i, lane, da[i]);
    }
    delta[0] = sdelta[warp * 16 + g8];
    delta[1] = sdelta[warp * 16 + g8 + 8];
    for (int kt = kt0; kt <= qt; ++kt) {
      const int buf = (kt - kt0) & 1;
      cp_async_wait<0>();
      __syncthreads();
      if (kt < qt) {
        load_tile<D, kT, kThreads>(sk + (buf ^ 1) * TB, k, p.k_ss, (kt + 1) * kT, pad, S, tid);
        load_tile<D, kT, kThreads>(sv + (buf ^ 1) * TB, v, p.v_ss, (kt + 1) * kT, pad, S, tid);
        cp_async_commit();
      }
      float s[8][4], dp[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = dp[j][e] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t bb[4];
          frag_b<D>(sk + buf * TB, 16 * j, 2 * i, lane, bb);
          mma16816<BF16>(s[2 * j], qa[i], bb[0], bb[1]);
          mma16816<BF16>(s[2 * j + 1], qa[i], bb[2], bb[3]);
          frag_b<D>(sv + buf * TB, 16 * j, 2 * i, lane, bb);
          mma16816<BF16>(dp[2 * j], da[i], bb[0], bb[1]);
          mma16816<BF16>(dp[2 * j + 1], da[i], bb[2], bb[3]);
        }
      if (kt == qt || kt * kT < pad) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kk = kt * kT + 8 * j + 2 * t4 + (e & 1), qq = q0 + warp * 16 + g8 + (e >> 1) * 8;
            if (kk > qq || kk < pad) s[j][e] = -INFINITY;
          }
      }
      if constexpr (DROP) {
        const uint32_t keep = keep_rows(key, blk + (unsigned)kt * (kT / 8), per_row, lane, p.threshold);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t bits = __shfl_sync(0xffffffffu, keep, g8 + 8 * r + (j >> 2) * 16) >> ((j & 3) * 8 + 2 * t4);
            dp[j][2 * r] = bits & 1u ? dp[j][2 * r] * p.inv_keep : 0.f;
            dp[j][2 * r + 1] = bits & 2u ? dp[j][2 * r + 1] * p.inv_keep : 0.f;
          }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = ex2_approx(fmaf(s[j][e], c2, -ls[e >> 1]));
      if (one_tile) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float d = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) d = fmaf(s[j][2 * r], dp[j][2 * r], fmaf(s[j][2 * r + 1], dp[j][2 * r + 1], d));
          d += __shfl_xor_sync(0xffffffffu, d, 1);
          d += __shfl_xor_sync(0xffffffffu, d, 2);
          delta[r] = d;
          const int row = q0 + warp * 16 + g8 + 8 * r;
          if (t4 == 0 && row < S) p.delta[row0 + row] = d;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] *= dp[j][e] - delta[e >> 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a[4] = {E::from_f2(s[2 * j][0], s[2 * j][1]), E::from_f2(s[2 * j][2], s[2 * j][3]),
                               E::from_f2(s[2 * j + 1][0], s[2 * j + 1][1]),
                               E::from_f2(s[2 * j + 1][2], s[2 * j + 1][3])};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t bb[4];
          frag_bt<D>(sk + buf * TB, 16 * j, 2 * i, lane, bb);
          mma16816<BF16>(acc[2 * i], a, bb[0], bb[1]);
          mma16816<BF16>(acc[2 * i + 1], a, bb[2], bb[3]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = q0 + warp * 16 + g8 + 8 * r;
    if (row >= S) continue;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<uint32_t*>(dq + row * p.dq_ss + 8 * i + 2 * t4) =
          E::from_f2(acc[i][2 * r] * p.scale, acc[i][2 * r + 1] * p.scale);
  }
}

// dk and dv of 64 keys of one KV head, over the R query heads that share it.
// The products are formed transposed (keys as rows), so P^T and dS^T are the
// left operands of dV and dK where they stand in registers.
template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kThreads) attn_train_dkv_kernel(const AttnTrainParams p, int ntiles) {
  constexpr int TB = kT * D * 2;
  __shared__ __align__(1024) uint8_t smem[4 * TB];
  __shared__ float slse[2][kT], sdelta[2][kT];
  const uint32_t sq = smem_u32(smem), sd = sq + 2 * TB;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int kt = (int)(blockIdx.x % (unsigned)ntiles);
  const unsigned bg = blockIdx.x / (unsigned)ntiles;
  const int b = (int)(bg / (unsigned)p.Hkv), g = (int)(bg % (unsigned)p.Hkv);
  const int S = p.S, k0 = kt * kT;
  const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), S) : 0;
  uint16_t* dk = static_cast<uint16_t*>(p.dk) + b * p.dk_sb + g * p.dk_sh;
  uint16_t* dv = static_cast<uint16_t*>(p.dv) + b * p.dv_sb + g * p.dv_sh;
  using E = Elem<BF16>;

  float ak[D / 8][4], av[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) ak[i][e] = av[i][e] = 0.f;

  if (min(S, k0 + kT) > pad) {
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + b * p.k_sb + g * p.k_sh;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.v_sb + g * p.v_sh;
    const float c2 = p.scale * 1.4426950408889634f;
    const int nq = ntiles - kt, items = nq * p.R;  // (head of the group, query tile) pairs, tiles fastest
    // K and V pass through the second buffers into registers.
    load_tile<D, kT, kThreads>(sq + TB, k, p.k_ss, k0, pad, S, tid);
    load_tile<D, kT, kThreads>(sd + TB, v, p.v_ss, k0, pad, S, tid);
    auto fetch = [&](int item, int buf) {
      const int h = g * p.R + item / nq, q0 = (kt + item % nq) * kT;
      load_tile<D, kT, kThreads>(sq + buf * TB, static_cast<const uint16_t*>(p.q) + b * p.q_sb + h * p.q_sh, p.q_ss, q0,
                                 pad, S, tid);
      load_tile<D, kT, kThreads>(sd + buf * TB, static_cast<const uint16_t*>(p.dout) + b * p.do_sb + h * p.do_sh,
                                 p.do_ss, q0, pad, S, tid);
      cp_async_commit();
      if (tid < kT) {
        const int row = q0 + tid;
        const long long at = ((long long)b * p.Hq + h) * S + row;
        const bool ok = row < S && row >= pad;
        slse[buf][tid] = ok ? __ldg(p.lse + at) : INFINITY;
        sdelta[buf][tid] = ok ? __ldg(p.delta + at) : 0.f;
      }
    };
    fetch(0, 0);
    DropKey key{};
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    if constexpr (DROP) key = drop_key(p.rng, p.site);
    cp_async_wait<0>();
    __syncthreads();
    uint32_t ka[D / 16][4], va[D / 16][4];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      frag_a<D>(sq + TB, warp * 16, 2 * i, lane, ka[i]);
      frag_a<D>(sd + TB, warp * 16, 2 * i, lane, va[i]);
    }
    for (int item = 0; item < items; ++item) {
      const int buf = item & 1;
      const int qt = kt + item % nq, q0 = qt * kT;
      cp_async_wait<0>();
      __syncthreads();
      if (item + 1 < items) fetch(item + 1, buf ^ 1);
      uint32_t keep = 0xffffffffu;
      if constexpr (DROP) {
        // Lane l: the two blocks of the warp's 16 keys in query rows l (low half) and l + 32 (high half).
        const unsigned h = (unsigned)(g * p.R + item / nq);
        const unsigned long long row = ((unsigned long long)b * (unsigned)p.Hq + h) * (unsigned)S + (unsigned)(q0 + lane);
        const unsigned long long blk = row * per_row + (unsigned)(k0 / 8 + warp * 2);
        const unsigned long long far = blk + 32ull * per_row;
        keep = keep_bits(key, blk, p.threshold) | keep_bits(key, blk + 1, p.threshold) << 8 |
               keep_bits(key, far, p.threshold) << 16 | keep_bits(key, far + 1, p.threshold) << 24;
      }
      const bool edge = qt == kt || k0 < pad;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float s[4][4], dp[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = dp[j][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t bb[4];
            frag_b<D>(sq + buf * TB, half * 32 + 16 * j, 2 * i, lane, bb);
            mma16816<BF16>(s[2 * j], ka[i], bb[0], bb[1]);
            mma16816<BF16>(s[2 * j + 1], ka[i], bb[2], bb[3]);
            frag_b<D>(sd + buf * TB, half * 32 + 16 * j, 2 * i, lane, bb);
            mma16816<BF16>(dp[2 * j], va[i], bb[0], bb[1]);
            mma16816<BF16>(dp[2 * j + 1], va[i], bb[2], bb[3]);
          }
        uint32_t pa[2][4], sa[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = half * 32 + 8 * j + 2 * t4;
          const float2 ls = *reinterpret_cast<const float2*>(&slse[buf][col]);
          const float2 dl = *reinterpret_cast<const float2*>(&sdelta[buf][col]);
          uint32_t bits0 = 0, bits1 = 0;
          if constexpr (DROP) {
            bits0 = __shfl_sync(0xffffffffu, keep, 8 * j + 2 * t4) >> (16 * half + g8);
            bits1 = __shfl_sync(0xffffffffu, keep, 8 * j + 2 * t4 + 1) >> (16 * half + g8);
          }
          float pd[4], ds[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float lq = e & 1 ? ls.y : ls.x, de = e & 1 ? dl.y : dl.x;
            float x = ex2_approx(fmaf(s[j][e], c2, -lq));
            float y = dp[j][e];
            bool single = false;
            if (edge) {
              const int kk = k0 + warp * 16 + g8 + (e >> 1) * 8, qq = q0 + col + (e & 1);
              if (kk > qq || kk < pad) x = 0.f;
              single = qq == pad;
            }
            pd[e] = x;
            if constexpr (DROP) {
              const bool stays = ((e & 1 ? bits1 : bits0) >> ((e >> 1) * 8)) & 1u;
              pd[e] = stays ? x : 0.f;
              y = stays ? y * p.inv_keep : 0.f;
            }
            ds[e] = single ? 0.f : x * (y - de);
          }
          pa[j >> 1][(j & 1) * 2] = E::from_f2(pd[0], pd[1]);
          pa[j >> 1][(j & 1) * 2 + 1] = E::from_f2(pd[2], pd[3]);
          sa[j >> 1][(j & 1) * 2] = E::from_f2(ds[0], ds[1]);
          sa[j >> 1][(j & 1) * 2 + 1] = E::from_f2(ds[2], ds[3]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t bb[4];
            frag_bt<D>(sd + buf * TB, half * 32 + 16 * j, 2 * i, lane, bb);
            mma16816<BF16>(av[2 * i], pa[j], bb[0], bb[1]);
            mma16816<BF16>(av[2 * i + 1], pa[j], bb[2], bb[3]);
            frag_bt<D>(sq + buf * TB, half * 32 + 16 * j, 2 * i, lane, bb);
            mma16816<BF16>(ak[2 * i], sa[j], bb[0], bb[1]);
            mma16816<BF16>(ak[2 * i + 1], sa[j], bb[2], bb[3]);
          }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = k0 + warp * 16 + g8 + 8 * r;
    if (row >= S) continue;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      *reinterpret_cast<uint32_t*>(dk + row * p.dk_ss + 8 * i + 2 * t4) =
          E::from_f2(ak[i][2 * r] * p.scale, ak[i][2 * r + 1] * p.scale);
      *reinterpret_cast<uint32_t*>(dv + row * p.dv_ss + 8 * i + 2 * t4) =
          E::from_f2(av[i][2 * r] * p.inv_keep, av[i][2 * r + 1] * p.inv_keep);
    }
  }
}

template <int D, bool BF16, bool DROP>
cudaError_t fwd(const AttnTrainParams& p, cudaStream_t st) {
  const int nt = (p.S + kT - 1) / kT;
  attn_train_fwd_kernel<D, BF16, DROP><<<(unsigned)((long long)nt * p.B * p.Hq), kThreads, 0, st>>>(p, nt);
  return cudaGetLastError();
}
template <int D, bool BF16, bool DROP>
cudaError_t bwd(const AttnTrainParams& p, cudaStream_t st) {
  const int nt = (p.S + kT - 1) / kT;
  attn_train_dq_kernel<D, BF16, DROP><<<(unsigned)((long long)nt * p.B * p.Hq), kThreads, 0, st>>>(p, nt);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  attn_train_dkv_kernel<D, BF16, DROP><<<(unsigned)((long long)nt * p.B * p.Hkv), kThreads, 0, st>>>(p, nt);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_train_fwd_sm100(const AttnTrainParams& p, int D, bool bf16, int num_sms, cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? fwd<32, true, true>(p, st) : fwd<32, true, false>(p, st))
                : (drop ? fwd<32, false, true>(p, st) : fwd<32, false, false>(p, st));
  return bf16 ? (drop ? fwd<64, true, true>(p, st) : fwd<64, true, false>(p, st))
              : (drop ? fwd<64, false, true>(p, st) : fwd<64, false, false>(p, st));
}

cudaError_t launch_attn_train_bwd_sm100(const AttnTrainParams& p, int D, bool bf16, int num_sms, cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? bwd<32, true, true>(p, st) : bwd<32, true, false>(p, st))
                : (drop ? bwd<32, false, true>(p, st) : bwd<32, false, false>(p, st));
  return bf16 ? (drop ? bwd<64, true, true>(p, st) : bwd<64, true, false>(p, st))
              : (drop ? bwd<64, false, true>(p, st) : bwd<64, false, false>(p, st));
}

}  // namespace dtk
