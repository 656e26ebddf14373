// Causal grouped-query attention for training on the tcgen05 tensor cores: the
// forward pass and the two passes of its gradient (formulas and roundings:
// attn_train_sm100.cu's head).
//
// Geometry.  Positions are counted from the first unpadded one: tiles of query
// rows and of keys start at `pad`, so padding costs nothing and is never read
// (a padded row's NaN times a zero weight would be a NaN).  A tile of query rows
// packs (position, head) pairs of the HC query heads that share a KV head (head
// fastest), so a group's K and V are fetched once and a short sequence still
// fills the 128 rows of an MMA; HC = R up to 64 heads, else chunks of 64.
//
// One CTA owns one tile and walks the other axis in blocks of 64, two or three
// CTAs per SM: while one CTA's threads turn scores into weights, another's
// products run.  Per block, with one thread issuing TMA and MMA (control warp)
// and the rest, one thread per row (forward) or two (backward), on the
// element-wise part:
//   forward   S = Q K^T             P -> TMEM, O += P V
//   dq        S = Q K^T, dP = dO V^T    dS -> TMEM, dQ += dS K
//   dk, dv    S^T = K Q^T, dP^T = V dO^T    P^T, dS^T -> TMEM, dV += P^T dO, dK += dS^T Q
// The left operand of every second product is written back into tensor memory
// over the scores that it came from; the right one is the shared-memory tile as
// TMA left it, read row-major ("MN major").  MMAs of one thread execute in
// order, so a block's scores may be issued behind the products that still read
// the previous block's weights in the same columns, and the commit of the
// scores also says that those products are done with their shared memory.
//
// What bounds it: an MMA of N = 64 costs about 50 cycles whatever its K, so at
// head_dim 64 a 128 x 64 block takes 400 (forward), 600 (dq) and 800 (dk, dv)
// tensor cycles, about as long as its element-wise part.
#include "attn_train_common.cuh"

namespace dtk {

namespace {

constexpr int kRows = 128;   // rows of a tile
constexpr int kBlk = 64;     // rows of a block of the other axis
constexpr int kStages = 2;   // blocks in flight
constexpr int kGroupUnits = 128;  // units scheduled together (their K / V stay in L2)

template <int D>
struct TcShape {
  static constexpr int ROWB = D * 2;
  static constexpr uint32_t LAYOUT = D == 64 ? kSw128 : kSw64;
  static constexpr int SBO = 8 * ROWB;
  static constexpr int TILE = kRows * ROWB;
  static constexpr int BLK = kBlk * ROWB;
  static constexpr int NCH = ROWB / 16;
};

// Barriers and small shared state behind the tiles.
struct TcShared {
  uint64_t tile_full, blk_full[kStages], s_full, p_full, o_full, drain;
  uint32_t tmem;
  int abort;
};

// Item i of the grid: units in groups, inside a group the tiles with the most
// work first.  longest_last: the last tile of a unit has the most blocks.
struct TcItem {
  int unit, tile;
};
__device__ __forceinline__ TcItem tc_item(long long i, int n_units, int tiles, bool longest_last) {
  const long long per = (long long)kGroupUnits * tiles;
  const int grp = (int)(i / per);
  const int j = (int)(i - grp * per);
  const int gu = min(kGroupUnits, n_units - grp * kGroupUnits);
  const int t = j / gu;
  return TcItem{grp * kGroupUnits + (j - t * gu), longest_last ? tiles - 1 - t : t};
}

// A unit: sample b, KV head g, and the chunk of HC query heads from h0 on.
struct TcUnit {
  int b, g, h0, heads, pad;
};
__device__ __forceinline__ TcUnit tc_unit(const AttnTrainParams& p, int unit, int chunks) {
  TcUnit u;
  const int bg = unit / chunks, c = unit - bg * chunks;
  u.b = bg / p.Hkv;
  u.g = bg - u.b * p.Hkv;
  u.h0 = u.g * p.R + c * p.HC;
  u.heads = min(p.HC, p.R - c * p.HC);
  u.pad = p.pad_len ? min(max(__ldg(p.pad_len + u.b), 0), p.S) : 0;
  return u;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status));
}

// Keep bits of 32 columns from `col` on of a dropout row (block index of the row's first block).
__device__ __forceinline__ uint32_t keep32(const DropKey& key, unsigned long long row_block, int col,
                                           uint32_t threshold) {
  const int shift = col & 7;
  const unsigned long long b = row_block + (unsigned)(col >> 3);
  uint32_t lo = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) lo |= keep_bits(key, b + i, threshold) << (8 * i);
  return shift ? __funnelshift_r(lo, keep_bits(key, b + 4, threshold), shift) : lo;
}

// Zeros rows [rows, total) of `count` tiles of `bytes` bytes each (the rows that
// TMA never fills when the packed heads leave some over).
template <int ROWB>
__device__ __forceinline__ void zero_rows(uint8_t* tiles, int count, int bytes, int rows, int total, int tid,
                                          int threads) {
  const int per = (total - rows) * (ROWB / 16);
  for (int e = tid; e < count * per; e += threads) {
    const int t = e / per, rem = e - t * per;
    *reinterpret_cast<uint4*>(tiles + t * bytes + rows * ROWB + rem * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Eight fp32 values, scaled, as 16 bytes.
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const uint32_t* v, float f) {
  using E = Elem<BF16>;
  return make_uint4(E::from_f2(__uint_as_float(v[0]) * f, __uint_as_float(v[1]) * f),
                    E::from_f2(__uint_as_float(v[2]) * f, __uint_as_float(v[3]) * f),
                    E::from_f2(__uint_as_float(v[4]) * f, __uint_as_float(v[5]) * f),
                    E::from_f2(__uint_as_float(v[6]) * f, __uint_as_float(v[7]) * f));
}

// Scores of one tile against one block: D[128 x 64] = A[128 x D] B[64 x D]^T.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) umma_f16_ss(tmem_d, a + 2 * kk, b + 2 * kk, idesc, kk > 0 ? 1u : 0u);
}
// D[128 x D] += A[128 x 64] B[64 x D] with A in tensor memory: columns 0 .. 15 hold
// its first 32 columns, 32 .. 47 the others (each half lies over its own scores).
template <int D>
__device__ __forceinline__ void issue_weights(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc,
                                              bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kBlk / 16; ++kk)
    umma_f16_ts(tmem_d, tmem_a + (uint32_t)((kk >> 1) * 32 + (kk & 1) * 8),
                b + (uint64_t)(kk * 16 * TcShape<D>::ROWB >> 4), idesc, (accumulate || kk > 0) ? 1u : 0u);
}

__device__ __forceinline__ void tc_init(TcShared* sh, int p_arrivals) {
  mbar_init(&sh->tile_full, 1);
  for (int i = 0; i < kStages; ++i) mbar_init(&sh->blk_full[i], 1);
  mbar_init(&sh->s_full, 1);
  mbar_init(&sh->p_full, p_arrivals);
  mbar_init(&sh->o_full, 1);
  mbar_init(&sh->drain, 1);
  sh->abort = 0;
  fence_mbar_init();
}

// ---------------------------------------------------------------- forward
constexpr int kFwdThreads = 160;

template <int D>
struct FwdSmem {
  using SH = TcShape<D>;
  static constexpr int OFF_K = SH::TILE;
  static constexpr int OFF_V = OFF_K + kStages * SH::BLK;
  static constexpr int OFF_SH = OFF_V + kStages * SH::BLK;
  static constexpr int NEED = OFF_SH + (int)sizeof(TcShared) + 1024;
  // At least a quarter of the SM's shared memory: four CTAs' 128 columns fill its tensor memory.
  static constexpr int BYTES = NEED > 50 * 1024 ? NEED : 50 * 1024;
};

template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kFwdThreads, 3)
    attn_train_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                             const __grid_constant__ CUtensorMap tmV, const AttnTrainParams p, int n_units, int chunks,
                             int tiles) {
  using SH = TcShape<D>;
  using SM = FwdSmem<D>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TcItem it = tc_item(blockIdx.x, n_units, tiles, true);
  const TcUnit u = tc_unit(p, it.unit, chunks);
  const int S = p.S, PT = kRows / p.HC, rows = PT * p.HC;
  const int p0 = u.pad + it.tile * PT;
  const bool work = p0 < S;
  const int nblk = work ? (min(p0 + PT, S) - 1 - u.pad) / kBlk + 1 : 0;

  if (work) {
    if (tid == 0) tc_init(sh, 4);
    if (warp == 4) {
      tmem_alloc(&sh->tmem, 128);
      tmem_relinquish();
    }
    zero_rows<SH::ROWB>(smem, 1, SH::TILE, rows, kRows, tid, kFwdThreads);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t t_s = sh->tmem, t_o = sh->tmem + 64;
    volatile int* abort = &sh->abort;

    if (warp == 4) {
      if (lane == 0) {
        const uint64_t qd = umma_smem_desc(smem_u32(smem), 16, SH::SBO, SH::LAYOUT);
        const uint64_t kd = umma_smem_desc(smem_u32(smem + SM::OFF_K), 16, SH::SBO, SH::LAYOUT);
        const uint64_t vd = umma_smem_desc(smem_u32(smem + SM::OFF_V), SH::BLK, SH::SBO, SH::LAYOUT);
        const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
        auto load = [&](int j) {
          const int st = j % kStages;
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * SH::BLK);
          tma_load_4d(smem + SM::OFF_K + st * SH::BLK, &tmK, &sh->blk_full[st], 0, u.g, u.pad + j * kBlk, u.b);
          tma_load_4d(smem + SM::OFF_V + st * SH::BLK, &tmV, &sh->blk_full[st], 0, u.g, u.pad + j * kBlk, u.b);
        };
        mbar_arrive_expect_tx(&sh->tile_full, (uint32_t)(rows * SH::ROWB));
        tma_load_4d(smem, &tmQ, &sh->tile_full, 0, u.h0, p0, u.b);
        int loaded = 0;
        for (; loaded < min(kStages, nblk); ++loaded) load(loaded);
        bool ok = mbar_wait(&sh->tile_full, 0, abort, p.status);
        for (int j = 0; j < nblk && ok; ++j) {
          const int st = j % kStages;
          const uint64_t at = (uint64_t)((st * SH::BLK) >> 4);
          if (!(ok = mbar_wait(&sh->blk_full[st], (j / kStages) & 1, abort, p.status))) break;
          tc_fence_after();
          issue_scores<D>(t_s, qd, kd + at, id_s);
          umma_commit(&sh->s_full);
          if (j > 0 && loaded < nblk) {
            // These scores being done, so is the previous block's P V: its stage is free.
            if (!(ok = mbar_wait(&sh->s_full, j & 1, abort, p.status))) break;
            load(loaded++);
          }
          if (!(ok = mbar_wait(&sh->p_full, j & 1, abort, p.status))) break;
          tc_fence_after();
          issue_weights<D>(t_o, t_s, vd + at, id_o, j > 0);
        }
        umma_commit(&sh->o_full);
        umma_commit(&sh->drain);
        mbar_wait(&sh->drain, 0, nullptr, nullptr);
        if (!ok) {
          // Copies still in flight must land before the CTA may end.
          mbar_wait(&sh->tile_full, 0, nullptr, nullptr);
          for (int j = max(0, loaded - kStages); j < loaded; ++j)
            mbar_wait(&sh->blk_full[j % kStages], (j / kStages) & 1, nullptr, nullptr);
        }
      }
      __syncwarp();
    } else {
      const int r = tid, head = r % p.HC, pos = p0 + r / p.HC;
      const bool valid = r < rows && head < u.heads && pos < S;
      const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
      const uint32_t ts = t_s + lane_off, to = t_o + lane_off;
      const float c2 = p.scale * 1.4426950408889634f;
      const long long row = ((long long)u.b * p.Hq + u.h0 + head) * S + pos;
      DropKey key{};
      unsigned long long row_block = 0;
      if constexpr (DROP) {
        key = drop_key(p.rng, p.site);
        row_block = (unsigned long long)row * ((unsigned)(S + 7) >> 3);
      }
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < nblk; ++j) {
        if (!(ok = warp_wait(&sh->s_full, j & 1, abort, p.status))) break;
        tc_fence_after();
        const int k0 = u.pad + j * kBlk;
        // Keys of the block that the row sees (a row without a query sees them all: it is not stored).
        const int see = valid ? pos - k0 + 1 : kBlk;
        uint32_t s0[32], s1[32];
        tmem_ld32_async(ts, s0);
        tmem_ld32_async(ts + 32, s1);
        tmem_wait_ld(s0);
        tmem_wait_ld(s1);
        if (__any_sync(0xffffffffu, see < kBlk)) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i >= see) s0[i] = 0xff800000u;
            if (i + 32 >= see) s1[i] = 0xff800000u;
          }
        }
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          x0 = fmax3(x0, __uint_as_float(s0[i]), __uint_as_float(s0[i + 1]));
          x1 = fmax3(x1, __uint_as_float(s1[i]), __uint_as_float(s1[i + 1]));
        }
        const float top = fmaxf(x0, x1) * c2;
        // The reference maximum moves only when a weight would pass 2^8; then O and l are
        // scaled by an exact power of two (P <= 256 is as exact in 16 bits as P <= 1).
        float f = 1.f;
        if (m == -INFINITY) {
          m = top;
        } else if (top > m + 8.f) {
          const float k = ceilf(top - m);
          m += k;
          f = exp2f(-k);
          l *= f;
        }
        if (__any_sync(0xffffffffu, f != 1.f)) {
          // This block's scores being done, so is the previous P V: O may be rewritten.
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16_u(to + c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(to + c, o);
          }
        }
        const float mm = m == -INFINITY ? 0.f : m;
        const float2 c2v = make_float2(c2, c2), nm = make_float2(-mm, -mm);
        auto half = [&](uint32_t (&s)[32], int c) {
          float2 sum = make_float2(0.f, 0.f);
          uint32_t pk[16];
          uint32_t keep = 0xffffffffu;
          if constexpr (DROP) keep = keep32(key, row_block, k0 + 32 * c, p.threshold);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 t = ffma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2v, nm);
            float2 w = make_float2(ex2_approx(t.x), ex2_approx(t.y));
            sum = fadd2(sum, w);
            if constexpr (DROP) {
              w.x = (keep >> i) & 1u ? w.x : 0.f;
              w.y = (keep >> (i + 1)) & 1u ? w.y : 0.f;
            }
            pk[i >> 1] = E::from_f2(w.x, w.y);
          }
          l += sum.x + sum.y;
          tmem_st16(ts + 32 * c, pk);
        };
        half(s0, 0);
        if (__any_sync(0xffffffffu, see > 32)) {
          half(s1, 1);
        } else {
          uint32_t z[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0u;
          tmem_st16(ts + 32, z);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      if (ok && warp_wait(&sh->o_full, 0, abort, p.status)) {
        tc_fence_after();
        uint32_t o[D];
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t(&part)[32] = *reinterpret_cast<uint32_t(*)[32]>(o + c);
          tmem_ld32_async(to + c, part);
          tmem_wait_ld(part);
        }
        if (valid) {
          const float inv = p.inv_keep / l;
          uint16_t* out = static_cast<uint16_t*>(p.o) + u.b * p.o_sb + (long long)pos * p.o_ss + (u.h0 + head) * p.o_sh;
#pragma unroll
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + c) = pack8<BF16>(o + c, inv);
          p.lse[row] = m + log2f(l);
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
      tc_fence_after();
      tmem_dealloc(sh->tmem, 128);
    }
  }
  // This tile's share of the padded rows: zeros.
  const int z0 = it.tile * PT, z1 = min(z0 + PT, u.pad);
  for (int e = tid; e < (z1 - z0) * u.heads * SH::NCH; e += kFwdThreads) {
    const int c = e % SH::NCH, rr = e / SH::NCH, head = u.h0 + rr % u.heads, pos = z0 + rr / u.heads;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + u.b * p.o_sb + (long long)pos * p.o_ss + head * p.o_sh +
                              c * 8) = make_uint4(0u, 0u, 0u, 0u);
    if (c == 0) p.lse[((long long)u.b * p.Hq + head) * S + pos] = INFINITY;
  }
}

// ---------------------------------------------------------------- dq
constexpr int kBwdThreads = 288;  // two element-wise warpgroups (half of a block's columns each) and the control warp

template <int D>
struct BwdSmem {
  using SH = TcShape<D>;
  static constexpr int OFF_B = SH::TILE;                    // second tile
  static constexpr int OFF_C = 2 * SH::TILE;                // first ring
  static constexpr int OFF_E = OFF_C + kStages * SH::BLK;   // second ring
  static constexpr int OFF_X = OFF_E + kStages * SH::BLK;   // 4 KB of rows' scalars
  static constexpr int OFF_SH = OFF_X + 4096;
  static constexpr int NEED = OFF_SH + (int)sizeof(TcShared) + 1024;
  // Above a third of the SM's shared memory: two CTAs' 256 columns fill its tensor memory.
  static constexpr int BYTES = NEED > 78 * 1024 ? NEED : 78 * 1024;
};

template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kBwdThreads, 2)
    attn_train_dq_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                            const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const AttnTrainParams p, int n_units, int chunks, int tiles) {
  using SH = TcShape<D>;
  using SM = BwdSmem<D>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  float* xrow = reinterpret_cast<float*>(smem + SM::OFF_X);  // [2][128] halves of delta
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TcItem it = tc_item(blockIdx.x, n_units, tiles, true);
  const TcUnit u = tc_unit(p, it.unit, chunks);
  const int S = p.S, PT = kRows / p.HC, rows = PT * p.HC;
  const int p0 = u.pad + it.tile * PT;
  const bool work = p0 < S;
  const int nblk = work ? (min(p0 + PT, S) - 1 - u.pad) / kBlk + 1 : 0;

  if (work) {
    if (tid == 0) tc_init(sh, 8);
    if (warp == 8) {
      tmem_alloc(&sh->tmem, 256);
      tmem_relinquish();
    }
    zero_rows<SH::ROWB>(smem, 2, SH::TILE, rows, kRows, tid, kBwdThreads);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t t_s = sh->tmem, t_dp = sh->tmem + 64, t_dq = sh->tmem + 128;
    volatile int* abort = &sh->abort;

    if (warp == 8) {
      if (lane == 0) {
        const uint64_t qd = umma_smem_desc(smem_u32(smem), 16, SH::SBO, SH::LAYOUT);
        const uint64_t dd = umma_smem_desc(smem_u32(smem + SM::OFF_B), 16, SH::SBO, SH::LAYOUT);
        const uint64_t kd = umma_smem_desc(smem_u32(smem + SM::OFF_C), 16, SH::SBO, SH::LAYOUT);
        const uint64_t vd = umma_smem_desc(smem_u32(smem + SM::OFF_E), 16, SH::SBO, SH::LAYOUT);
        const uint64_t kt = umma_smem_desc(smem_u32(smem + SM::OFF_C), SH::BLK, SH::SBO, SH::LAYOUT);
        const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
        auto load = [&](int j) {
          const int st = j % kStages;
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * SH::BLK);
          tma_load_4d(smem + SM::OFF_C + st * SH::BLK, &tmK, &sh->blk_full[st], 0, u.g, u.pad + j * kBlk, u.b);
          tma_load_4d(smem + SM::OFF_E + st * SH::BLK, &tmV, &sh->blk_full[st], 0, u.g, u.pad + j * kBlk, u.b);
        };
        mbar_arrive_expect_tx(&sh->tile_full, 2u * (uint32_t)(rows * SH::ROWB));
        tma_load_4d(smem, &tmQ, &sh->tile_full, 0, u.h0, p0, u.b);
        tma_load_4d(smem + SM::OFF_B, &tmDO, &sh->tile_full, 0, u.h0, p0, u.b);
        int loaded = 0;
        for (; loaded < min(kStages, nblk); ++loaded) load(loaded);
        bool ok = mbar_wait(&sh->tile_full, 0, abort, p.status);
        for (int j = 0; j < nblk && ok; ++j) {
          const int st = j % kStages;
          const uint64_t at = (uint64_t)((st * SH::BLK) >> 4);
          if (!(ok = mbar_wait(&sh->blk_full[st], (j / kStages) & 1, abort, p.status))) break;
          tc_fence_after();
          issue_scores<D>(t_s, qd, kd + at, id_s);
          issue_scores<D>(t_dp, dd, vd + at, id_s);
          umma_commit(&sh->s_full);
          if (j > 0 && loaded < nblk) {
            if (!(ok = mbar_wait(&sh->s_full, j & 1, abort, p.status))) break;
            load(loaded++);
          }
          if (!(ok = mbar_wait(&sh->p_full, j & 1, abort, p.status))) break;
          tc_fence_after();
          issue_weights<D>(t_dq, t_s, kt + at, id_o, j > 0);
        }
        umma_commit(&sh->o_full);
        umma_commit(&sh->drain);
        mbar_wait(&sh->drain, 0, nullptr, nullptr);
        if (!ok) {
          mbar_wait(&sh->tile_full, 0, nullptr, nullptr);
          for (int j = max(0, loaded - kStages); j < loaded; ++j)
            mbar_wait(&sh->blk_full[j % kStages], (j / kStages) & 1, nullptr, nullptr);
        }
      }
      __syncwarp();
    } else {
      const int half = warp >> 2, wq = warp & 3, r = wq * 32 + lane;
      const int head = r % p.HC, pos = p0 + r / p.HC;
      const bool valid = r < rows && head < u.heads && pos < S;
      const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
      const uint32_t ts = t_s + lane_off + 32 * half, tdp = t_dp + lane_off + 32 * half;
      const float c2 = p.scale * 1.4426950408889634f;
      const long long row = ((long long)u.b * p.Hq + u.h0 + head) * S + pos;
      // A row with a single key (pos == pad) has no gradient: its P is taken as 0.
      const float ls = valid && pos != u.pad ? __ldg(p.lse + row) : INFINITY;
      DropKey key{};
      unsigned long long row_block = 0;
      if constexpr (DROP) {
        key = drop_key(p.rng, p.site);
        row_block = (unsigned long long)row * ((unsigned)(S + 7) >> 3);
      }
      float delta = 0.f;
      bool ok = true;
      if (nblk > 1) {
        // delta = O . dO: each of the row's two threads takes half of the columns.
        uint4 o[SH::NCH / 2];
        const uint16_t* po = static_cast<const uint16_t*>(p.o) + u.b * p.o_sb + (long long)pos * p.o_ss +
                             (u.h0 + head) * p.o_sh + half * (D / 2);
#pragma unroll
        for (int i = 0; i < SH::NCH / 2; ++i)
          o[i] = valid ? __ldg(reinterpret_cast<const uint4*>(po) + i) : make_uint4(0u, 0u, 0u, 0u);
        if ((ok = warp_wait(&sh->tile_full, 0, abort, p.status))) {
          float d = 0.f;
#pragma unroll
          for (int i = 0; i < SH::NCH / 2; ++i) {
            const uint4 g = *reinterpret_cast<const uint4*>(smem + SM::OFF_B +
                                                            swz<SH::ROWB>(r, half * (SH::NCH / 2) + i));
            const uint32_t a[4] = {o[i].x, o[i].y, o[i].z, o[i].w}, c[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 x = E::to_f2(a[e]), y = E::to_f2(c[e]);
              d = fmaf(x.x, y.x, fmaf(x.y, y.y, d));
            }
          }
          xrow[half * kRows + r] = d;
        }
        ok = named_bar_and(1, 256, ok);
        if (ok) {
          delta = xrow[r] + xrow[kRows + r];
          if (half == 0 && valid) p.delta[row] = delta;
        }
      }
      for (int j = 0; j < nblk && ok; ++j) {
        if (!(ok = warp_wait(&sh->s_full, j & 1, abort, p.status))) {
          if (nblk == 1) named_bar_and(1, 256, false);
          break;
        }
        tc_fence_after();
        const int k0 = u.pad + j * kBlk + 32 * half;
        const int see = valid ? pos - k0 + 1 : 32;
        uint32_t s[32], dp[32];
        tmem_ld32_async(ts, s);
        tmem_ld32_async(tdp, dp);
        tmem_wait_ld(s);
        tmem_wait_ld(dp);
        uint32_t keep = 0xffffffffu;
        if constexpr (DROP) {
          if (__any_sync(0xffffffffu, see > 0)) keep = keep32(key, row_block, k0, p.threshold);
        }
        const bool masked = __any_sync(0xffffffffu, see < 32);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float w = ex2_approx(fmaf(__uint_as_float(s[i]), c2, -ls));
          if (masked && i >= see) w = 0.f;
          float d = __uint_as_float(dp[i]);
          if constexpr (DROP) d = (keep >> i) & 1u ? d * p.inv_keep : 0.f;
          s[i] = __float_as_uint(w);
          dp[i] = __float_as_uint(d);
        }
        if (nblk == 1) {
          // All keys of these rows are here: delta from the unrounded terms.
          float d = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) d = fmaf(__uint_as_float(s[i]), __uint_as_float(dp[i]), d);
          xrow[half * kRows + r] = d;
          if (!(ok = named_bar_and(1, 256, true))) break;
          delta = xrow[r] + xrow[kRows + r];
          if (half == 0 && valid) p.delta[row] = delta;
        }
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          pk[i >> 1] = E::from_f2(__uint_as_float(s[i]) * (__uint_as_float(dp[i]) - delta),
                                  __uint_as_float(s[i + 1]) * (__uint_as_float(dp[i + 1]) - delta));
        tmem_st16(ts, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      if (ok && warp_wait(&sh->o_full, 0, abort, p.status)) {
        tc_fence_after();
        uint32_t o[D / 2];
#pragma unroll
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t(&part)[16] = *reinterpret_cast<uint32_t(*)[16]>(o + c);
          tmem_ld16_u(t_dq + lane_off + half * (D / 2) + c, part);
        }
        if (valid) {
          uint16_t* dq = static_cast<uint16_t*>(p.dq) + u.b * p.dq_sb + (long long)pos * p.dq_ss +
                         (u.h0 + head) * p.dq_sh + half * (D / 2);
#pragma unroll
          for (int c = 0; c < D / 2; c += 8) *reinterpret_cast<uint4*>(dq + c) = pack8<BF16>(o + c, p.scale);
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
      tc_fence_after();
      tmem_dealloc(sh->tmem, 256);
    }
  }
  const int z0 = it.tile * PT, z1 = min(z0 + PT, u.pad);
  for (int e = tid; e < (z1 - z0) * u.heads * SH::NCH; e += kBwdThreads) {
    const int c = e % SH::NCH, rr = e / SH::NCH, head = u.h0 + rr % u.heads, pos = z0 + rr / u.heads;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dq) + u.b * p.dq_sb + (long long)pos * p.dq_ss + head * p.dq_sh +
                              c * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ---------------------------------------------------------------- dk, dv
template <int D, bool BF16, bool DROP>
__global__ void __launch_bounds__(kBwdThreads, 2)
    attn_train_dkv_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                             const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                             const AttnTrainParams p, int n_units, int chunks, int tiles) {
  using SH = TcShape<D>;
  using SM = BwdSmem<D>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TcItem it = tc_item(blockIdx.x, n_units, tiles, false);
  const int b = it.unit / p.Hkv, g = it.unit - b * p.Hkv;
  const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), p.S) : 0;
  const int S = p.S, PT = kBlk / p.HC, rows = PT * p.HC;
  const int k0 = pad + it.tile * kRows;
  const bool work = k0 < S;
  // Blocks of PT positions from k0 on (earlier queries see none of these keys) x chunks of heads.
  const int per = work ? (S - k0 + PT - 1) / PT : 0, nblk = per * chunks;

  if (work) {
    if (tid == 0) tc_init(sh, 8);
    if (warp == 8) {
      tmem_alloc(&sh->tmem, 256);
      tmem_relinquish();
    }
    zero_rows<SH::ROWB>(smem + SM::OFF_C, 2 * kStages, SH::BLK, rows, kBlk, tid, kBwdThreads);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t t_s = sh->tmem, t_dp = sh->tmem + 64, t_dv = sh->tmem + 128, t_dk = sh->tmem + 128 + D;
    volatile int* abort = &sh->abort;

    if (warp == 8) {
      if (lane == 0) {
        const uint64_t kd = umma_smem_desc(smem_u32(smem), 16, SH::SBO, SH::LAYOUT);
        const uint64_t vd = umma_smem_desc(smem_u32(smem + SM::OFF_B), 16, SH::SBO, SH::LAYOUT);
        const uint64_t qd = umma_smem_desc(smem_u32(smem + SM::OFF_C), 16, SH::SBO, SH::LAYOUT);
        const uint64_t dd = umma_smem_desc(smem_u32(smem + SM::OFF_E), 16, SH::SBO, SH::LAYOUT);
        const uint64_t qt = umma_smem_desc(smem_u32(smem + SM::OFF_C), SH::BLK, SH::SBO, SH::LAYOUT);
        const uint64_t dt = umma_smem_desc(smem_u32(smem + SM::OFF_E), SH::BLK, SH::SBO, SH::LAYOUT);
        const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
        auto load = [&](int j) {
          const int st = j % kStages, h0 = g * p.R + (j / per) * p.HC, q0 = k0 + (j % per) * PT;
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * (uint32_t)(rows * SH::ROWB));
          tma_load_4d(smem + SM::OFF_C + st * SH::BLK, &tmQ, &sh->blk_full[st], 0, h0, q0, b);
          tma_load_4d(smem + SM::OFF_E + st * SH::BLK, &tmDO, &sh->blk_full[st], 0, h0, q0, b);
        };
        mbar_arrive_expect_tx(&sh->tile_full, 2u * SH::TILE);
        tma_load_4d(smem, &tmK, &sh->tile_full, 0, g, k0, b);
        tma_load_4d(smem + SM::OFF_B, &tmV, &sh->tile_full, 0, g, k0, b);
        int loaded = 0;
        for (; loaded < min(kStages, nblk); ++loaded) load(loaded);
        bool ok = mbar_wait(&sh->tile_full, 0, abort, p.status);
        for (int j = 0; j < nblk && ok; ++j) {
          const int st = j % kStages;
          const uint64_t at = (uint64_t)((st * SH::BLK) >> 4);
          if (!(ok = mbar_wait(&sh->blk_full[st], (j / kStages) & 1, abort, p.status))) break;
          tc_fence_after();
          issue_scores<D>(t_s, kd, qd + at, id_s);
          issue_scores<D>(t_dp, vd, dd + at, id_s);
          umma_commit(&sh->s_full);
          if (j > 0 && loaded < nblk) {
            if (!(ok = mbar_wait(&sh->s_full, j & 1, abort, p.status))) break;
            load(loaded++);
          }
          if (!(ok = mbar_wait(&sh->p_full, j & 1, abort, p.status))) break;
          tc_fence_after();
          issue_weights<D>(t_dv, t_s, dt + at, id_o, j > 0);
          issue_weights<D>(t_dk, t_dp, qt + at, id_o, j > 0);
        }
        umma_commit(&sh->o_full);
        umma_commit(&sh->drain);
        mbar_wait(&sh->drain, 0, nullptr, nullptr);
        if (!ok) {
          mbar_wait(&sh->tile_full, 0, nullptr, nullptr);
          for (int j = max(0, loaded - kStages); j < loaded; ++j)
            mbar_wait(&sh->blk_full[j % kStages], (j / kStages) & 1, nullptr, nullptr);
        }
      }
      __syncwarp();
    } else {
      const int half = warp >> 2, wq = warp & 3, r = wq * 32 + lane;
      const int key0 = k0 + wq * 32, kk = key0 + lane;  // the warp's keys, the thread's
      const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
      const uint32_t ts = t_s + lane_off + 32 * half, tdp = t_dp + lane_off + 32 * half;
      const float c2 = p.scale * 1.4426950408889634f;
      DropKey key{};
      const unsigned per_row = (unsigned)(S + 7) >> 3;
      if constexpr (DROP) key = drop_key(p.rng, p.site);
      // Scalars of the warp's 32 columns (query rows): lane l fetches those of column l.
      float2* x_ld = reinterpret_cast<float2*>(smem + SM::OFF_X) + warp * 32;             // lse, delta
      uint32_t* x_keep = reinterpret_cast<uint32_t*>(smem + SM::OFF_X + 2048) + warp * 32;  // keep bits of the warp's keys
      int* x_pos = reinterpret_cast<int*>(smem + SM::OFF_X + 3072) + warp * 32;
      const int col = 32 * half + lane, chead = col % p.HC, cpos = col / p.HC;
      bool ok = true;
      for (int j = 0; j < nblk; ++j) {
        const int chunk = j / per, q0 = k0 + (j - chunk * per) * PT;
        const int pos = q0 + cpos;
        const bool valid = col < rows && chunk * p.HC + chead < p.R && pos < S;
        const long long row = ((long long)b * p.Hq + g * p.R + chunk * p.HC + chead) * S + pos;
        float2 ld = make_float2(INFINITY, 0.f);
        if (valid) ld = make_float2(__ldg(p.lse + row), __ldg(p.delta + row));
        uint32_t keep = 0;
        if constexpr (DROP) {
          if (valid && pos >= key0) keep = keep32(key, (unsigned long long)row * per_row, key0, p.threshold);
        }
        __syncwarp();
        x_ld[lane] = ld;
        if constexpr (DROP) x_keep[lane] = keep;
        x_pos[lane] = pos;
        __syncwarp();
        if (!(ok = warp_wait(&sh->s_full, j & 1, abort, p.status))) break;
        tc_fence_after();
        uint32_t s[32], dp[32];
        tmem_ld32_async(ts, s);
        tmem_ld32_async(tdp, dp);
        tmem_wait_ld(s);
        tmem_wait_ld(dp);
        // Only blocks on the diagonal hold queries before a key, and only the first the row with a single key.
        const bool edge = q0 < key0 + 31 || q0 == pad;
        uint32_t pw[16], pd[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float4 a = *reinterpret_cast<const float4*>(x_ld + i);  // lse, delta of two columns
          float w0 = ex2_approx(fmaf(__uint_as_float(s[i]), c2, -a.x));
          float w1 = ex2_approx(fmaf(__uint_as_float(s[i + 1]), c2, -a.z));
          float d0 = __uint_as_float(dp[i]), d1 = __uint_as_float(dp[i + 1]);
          float g0 = 1.f, g1 = 1.f;
          if (edge) {
            const int2 q = *reinterpret_cast<const int2*>(x_pos + i);
            if (kk > q.x) w0 = 0.f;
            if (kk > q.y) w1 = 0.f;
            if (q.x == pad) g0 = 0.f;
            if (q.y == pad) g1 = 0.f;
          }
          float v0 = w0, v1 = w1;
          if constexpr (DROP) {
            const uint2 kb = *reinterpret_cast<const uint2*>(x_keep + i);
            const bool y0 = (kb.x >> lane) & 1u, y1 = (kb.y >> lane) & 1u;
            v0 = y0 ? w0 : 0.f;
            v1 = y1 ? w1 : 0.f;
            d0 = y0 ? d0 * p.inv_keep : 0.f;
            d1 = y1 ? d1 * p.inv_keep : 0.f;
          }
          pw[i >> 1] = E::from_f2(v0, v1);
          d0 = w0 * (d0 - a.y);
          d1 = w1 * (d1 - a.w);
          if (edge) {
            d0 *= g0;
            d1 *= g1;
          }
          pd[i >> 1] = E::from_f2(d0, d1);
        }
        tmem_st16(ts, pw);
        tmem_st16(tdp, pd);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      if (ok && warp_wait(&sh->o_full, 0, abort, p.status)) {
        tc_fence_after();
        // The first warpgroup stores dv, the second dk.
        const uint32_t from = (half ? t_dk : t_dv) + lane_off;
        const float f = half ? p.scale : p.inv_keep;
        uint32_t o[D];
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t(&part)[32] = *reinterpret_cast<uint32_t(*)[32]>(o + c);
          tmem_ld32_async(from + c, part);
          tmem_wait_ld(part);
        }
        if (kk < S) {
          uint16_t* dst = half ? static_cast<uint16_t*>(p.dk) + b * p.dk_sb + (long long)kk * p.dk_ss + g * p.dk_sh
                               : static_cast<uint16_t*>(p.dv) + b * p.dv_sb + (long long)kk * p.dv_ss + g * p.dv_sh;
#pragma unroll
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(dst + c) = pack8<BF16>(o + c, f);
        }
      }
      (void)r;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
      tc_fence_after();
      tmem_dealloc(sh->tmem, 256);
    }
  }
  const int z0 = it.tile * kRows, z1 = min(z0 + kRows, pad);
  for (int e = tid; e < (z1 - z0) * SH::NCH; e += kBwdThreads) {
    const int c = e % SH::NCH, pos = z0 + e / SH::NCH;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dk) + b * p.dk_sb + (long long)pos * p.dk_ss + g * p.dk_sh +
                              c * 8) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dv) + b * p.dv_sb + (long long)pos * p.dv_ss + g * p.dv_sh +
                              c * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int D, bool BF16, bool DROP>
cudaError_t tc_fwd(const AttnTrainParams& p, const AttnTrainMaps& m, cudaStream_t st) {
  auto kern = attn_train_fwd_tc_kernel<D, BF16, DROP>;
  const cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kern), FwdSmem<D>::BYTES);
  if (e != cudaSuccess) return e;
  const int chunks = (p.R + p.HC - 1) / p.HC, units = p.B * p.Hkv * chunks, PT = kRows / p.HC;
  const int tiles = (p.S + PT - 1) / PT;
  kern<<<(unsigned)((long long)units * tiles), kFwdThreads, FwdSmem<D>::BYTES, st>>>(m.q_tile, m.k_blk, m.v_blk, p,
                                                                                     units, chunks, tiles);
  return cudaGetLastError();
}
template <int D, bool BF16, bool DROP>
cudaError_t tc_bwd(const AttnTrainParams& p, const AttnTrainMaps& m, cudaStream_t st) {
  auto kq = attn_train_dq_tc_kernel<D, BF16, DROP>;
  auto kk = attn_train_dkv_tc_kernel<D, BF16, DROP>;
  cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kq), BwdSmem<D>::BYTES);
  if (e != cudaSuccess) return e;
  if ((e = smem_limit_once(reinterpret_cast<const void*>(kk), BwdSmem<D>::BYTES)) != cudaSuccess) return e;
  const int chunks = (p.R + p.HC - 1) / p.HC, PT = kRows / p.HC;
  const int units = p.B * p.Hkv, tiles = (p.S + PT - 1) / PT, ktiles = (p.S + kRows - 1) / kRows;
  kq<<<(unsigned)((long long)units * chunks * tiles), kBwdThreads, BwdSmem<D>::BYTES, st>>>(
      m.q_tile, m.do_tile, m.k_blk, m.v_blk, p, units * chunks, chunks, tiles);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  kk<<<(unsigned)((long long)units * ktiles), kBwdThreads, BwdSmem<D>::BYTES, st>>>(m.k_tile, m.v_tile, m.q_blk,
                                                                                    m.do_blk, p, units, chunks, ktiles);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_train_fwd_tc_sm100(const AttnTrainParams& p, const AttnTrainMaps& m, int D, bool bf16,
                                           cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? tc_fwd<32, true, true>(p, m, st) : tc_fwd<32, true, false>(p, m, st))
                : (drop ? tc_fwd<32, false, true>(p, m, st) : tc_fwd<32, false, false>(p, m, st));
  return bf16 ? (drop ? tc_fwd<64, true, true>(p, m, st) : tc_fwd<64, true, false>(p, m, st))
              : (drop ? tc_fwd<64, false, true>(p, m, st) : tc_fwd<64, false, false>(p, m, st));
}

cudaError_t launch_attn_train_bwd_tc_sm100(const AttnTrainParams& p, const AttnTrainMaps& m, int D, bool bf16,
                                           cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? tc_bwd<32, true, true>(p, m, st) : tc_bwd<32, true, false>(p, m, st))
                : (drop ? tc_bwd<32, false, true>(p, m, st) : tc_bwd<32, false, false>(p, m, st));
  return bf16 ? (drop ? tc_bwd<64, true, true>(p, m, st) : tc_bwd<64, true, false>(p, m, st))
              : (drop ? tc_bwd<64, false, true>(p, m, st) : tc_bwd<64, false, false>(p, m, st));
}

}  // namespace dtk
