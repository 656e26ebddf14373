// Causal grouped-query attention for training, with its gradient, on the tcgen05
// tensor cores.
//
// For a query row q >= pad of head h (KV head g = h / R) and keys j in pad..q:
//   s_j = scale q . k_j,   P_j = exp(s_j) / sum exp,   O = sum_j m'_j P_j v_j
// with m' = m / (1 - p), m the dropout mask (philox.cuh).  Rows q < pad see no
// key: O = 0, no gradient.  Backward:
//   dV_j = sum_q m' P dO,   dP_j = m' dO . v_j,   delta = sum_j P_j dP_j = O . dO
//   dS_j = P_j (dP_j - delta),   dq = scale sum_j dS_j k_j,   dk_j = scale sum_q dS_j q
// The forward pass keeps log2 of each row's softmax denominator (base 2), so the
// backward passes form P again from one product.
//
// Two backward kernels: one walks the keys of a tile of query rows (delta, dq),
// one walks the query rows behind a tile of keys (dk, dv).  Each sum has one
// owner: no atomics, the same bits every run; the price is that S and dP are
// formed twice.  When the tiles are too few for the GPU, the other axis of each is
// dealt out to several CTAs, whose fp32 sums a further kernel joins in order.  The
// dropout mask of a block is generated by the dq kernel, which hands it on as bits
// (for contexts up to 64 positions for each of D; beyond, both generate it).
//
// Rounding: P and dS enter the second products in the inputs' 16-bit type, as
// the tensor cores take both operands in one type; sums, softmax statistics
// and delta are fp32.  fp16 has no exponents for P of long rows nor for dS of small
// gradients, so there both are scaled by powers of two, which the stores take out
// again: P of the dk, dv kernel by 2^15 (P <= 1), dS by a factor of its sample and KV
// head (GradExponent; forward, P is relative to a running maximum).  A row with a single key has a constant softmax: its dS
// is set to exactly zero.  Where a tile's keys are one block, delta is the sum
// over the unrounded P dP; beyond, it is O . dO with the stored O.
//
// Geometry.  A tile of 128 query rows packs (position, head) pairs of the HC
// query heads that share a KV head (head fastest), so a group's K and V are
// fetched once and a short sequence still fills an MMA; HC = R up to 64 heads,
// else chunks of 64.  Tiles of query rows start at the first unpadded position,
// blocks and tiles of keys at the multiple of 8 before it (where a block of the
// dropout generator starts): padding costs nothing, and the up to seven padded
// keys of a first block are zeroed in shared memory, so what stands there never
// meets a product (a NaN times a zero weight would be a NaN).
//
// Two CTAs on each SM, which take tile after tile until the launch has none left
// (claim_item).  One thread loads tiles and blocks by TMA, one
// issues the MMAs; the other warps are the element-wise part, one thread per row
// (forward) or two (backward).  Per block of 64:
//   forward   S = Q K^T             P -> TMEM, O += P V
//   dq        S = Q K^T, dP = dO V^T    dS -> TMEM, dQ += dS K
//   dk, dv    S^T = K Q^T, dP^T = V dO^T    P^T, dS^T -> TMEM, dV += P^T dO, dK += dS^T Q
// The left operand of every second product goes back to tensor memory, the
// right one is the shared-memory tile as TMA left it, read row-major ("MN
// major").  The next block's scores are issued as soon as this block's are in
// registers.  The weights have columns of their own, except for dk and dv with
// D = 64, where the columns do not hold both: there P^T lies over S^T and dS^T over
// dP^T.  For dk and dv the two halves of a block alternate: while the threads form
// dS^T of a block, dV += P^T dO and the next S^T run, and during the next
// exponentials dK += dS^T Q and the next dP^T.
//
// Order between MMAs.  The PTX ISA promises it for those of one accumulator and
// shape only.  So whatever is read by one MMA and written by another (weights that
// lie where the next scores go), or by the threads, is handed on through a commit and
// a wait on its mbarrier.
//
// What bounds it.  96 x 768, 12 / 4 heads of 64, padding up to half, bf16, p = 0.1:
// forward 214 us, dq 246, dk and dv 272 (0.18 PFLOP of products that count: 243
// TFLOP/s); half that batch without dropout 80, 93 and 138 us, with it 118, 136 and
// 166.  No unit is full: the tensor pipe is busy 20 to 27 % of the time without
// dropout (an MMA of N = 64 costs about 50 cycles whatever its K: 400, 600 and 800 for
// a 128 x 64 block), the exponentials' unit 21 to 39 %, and 41 to 47 % of the issue
// slots are used (with dropout 50 to 56 %: a generator call is 65 instructions for
// eight scores).  The dk, dv kernel spills 76 to 136 bytes a thread in most forms, and
// with D = 64 its scores' waits for the weights under them cost 132 -> 138 us of the
// case without dropout (164 -> 166 with it).  A block is a chain from the scores over tensor memory, the
// exponentials, tensor memory again and the next product, and two CTAs on an SM (four
// warps a scheduler in the backward kernels) cover each other's waits only in part.
// Four forward CTAs with a quarter of the columns each, the weights over the scores,
// were slower (307 us): their scores wait for the product before.
#include <utility>

#include "dt_common.cuh"
#include "dt_internal.h"
#include "philox.cuh"
#include "prefill_common.cuh"

namespace dtk {

namespace {

constexpr int kRows = 128;   // rows of a tile
constexpr int kBlk = 64;     // rows of a block of the other axis
// The dq kernel hands its drop flags on for up to this many positions per head
// dimension: S / 8 bytes a query row against 2 D of q itself, so at most four times q.
constexpr int kWordsPerDim = 64;
constexpr int kMaxStages = 4;
constexpr int kPerSm = 2;       // CTAs on an SM: each takes half of its tensor memory
constexpr uint32_t kCols = 256;
constexpr int kFwdBufs = 2;     // score buffers of the forward kernel
constexpr int kGroupUnits = 128;  // units scheduled together (their K / V stay in L2)

template <int D>
struct TcShape {
  static constexpr int ROWB = D * 2;
  static constexpr uint32_t LAYOUT = D == 64 ? kSw128 : kSw64;
  static constexpr int SBO = 8 * ROWB;
  static constexpr int TILE = kRows * ROWB;
  static constexpr int BLK = kBlk * ROWB;
  static constexpr int NCH = ROWB / 16;
  // Tile buffers of the backward kernels and blocks in flight: what the memory of two CTAs allows.
  static constexpr int BWD_TILES = D == 64 ? 1 : 2;
  static constexpr int DQ_STAGES = D == 64 ? 3 : 4;
  static constexpr int STAGES = 4;
};

// An item as the loading thread hands it to the element-wise warps.
constexpr int kItems = 8;
struct alignas(16) Item {
  int nblk, pad, heads, tile;  // blocks (-1: no more items); heads of the chunk
  int first, origin, per, split;  // rows: p0, kb; keys: q0, k0, blocks of a chunk of heads, the first block
  long long row;   // of lse, delta and the dropout rows: sample and first head, position 0
  int lift;        // exponent of dS's factor (fp16)
  long long out, out2, part;  // element offsets of the outputs at that sample and head, position 0; rows of partial sums
};

// Barriers and small shared state behind the tiles.
struct TcShared {
  uint64_t tile_full[2], tile_empty[2], blk_full[kMaxStages], blk_empty[kMaxStages];
  uint64_t s_full[2], s_read[2], dp_full, p_full, ds_full, w_done, o_empty, drain;
  uint64_t p_taken;  // dk, dv with the weights over the scores: P^T has been read
  uint64_t pair[4];  // dq: the two warps that share rows have both halves of delta in place
  uint64_t item_full[kItems], item_empty[kItems];
  Item item[kItems];  // the items under way
  alignas(16) uint4 claim[2];  // answers to the requests for items, in turn
  uint64_t claimed;
  int2 tile_meta[8];  // blocks and padded keys of the tiles under way (0 blocks: no more tiles)
  float inverse[8], out_scale[2][8];  // dq, fp16: 1 / dS's factor, and scale / factor of two items in turn; each warp's own
  uint32_t tmem;
  int abort;
};

// How a kernel's items are numbered: units in groups, inside a group the tiles
// with the most work first (longest_last: a unit's last tile has the most blocks).
struct Grid {
  int units, tiles, items, chunks, splits;  // chunks of a group's heads; CTAs that share a tile
  int seg;                                  // tiles of rows: key blocks of a segment
  FastDiv by_tiles, by_parts, by_kv;        // parts of a unit: chunks or splits (never both)
};
struct TcItem {
  int unit, tile;
};
__device__ __forceinline__ TcItem tc_item(const Grid& gr, int i, bool longest_last) {
  static_assert(kGroupUnits == 128, "shifts below");
  const int grp = gr.by_tiles(i >> 7);
  const int j = i - grp * (kGroupUnits * gr.tiles);
  const int gu = min(kGroupUnits, gr.units - grp * kGroupUnits);
  const int t = gu == kGroupUnits ? j >> 7 : j / gu;
  return TcItem{grp * kGroupUnits + (j - t * gu), longest_last ? gr.tiles - 1 - t : t};
}

// Takes an item: cancels the launch of the first CTA that has not started yet and
// returns its index, -1 when none is left (then no further request may follow) or, with
// ok false, when no answer came.  Items are of very different lengths (causality,
// padding), and a CTA that is done takes the next one of the whole launch: dealt out
// in turn beforehand, the busiest SM had 1.26 (dq) to 1.6 times (dk, dv) the mean's work.
__device__ __forceinline__ int claim_item(TcShared* sh, int n, volatile int* abort, int* status, bool& ok) {
  const uint32_t at = smem_u32(&sh->claim[n & 1]);
  fence_proxy_async_smem();  // behind this thread's earlier reads of the place
  mbar_arrive_expect_tx(&sh->claimed, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(at),
               "r"(smem_u32(&sh->claimed))
               : "memory");
  ok = mbar_wait(&sh->claimed, n & 1, abort, status);
  if (!ok) {
    mbar_wait(&sh->claimed, n & 1, nullptr, nullptr);  // the answer must not come behind the CTA's end
    return -1;
  }
  int got, index;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t"
      "mov.b32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, r;\n\t}"
      : "=r"(got), "=r"(index)
      : "r"(at)
      : "memory");
  return got ? index : -1;
}

// A tile of query rows: sample b, KV head g, the chunk of HC query heads from h0
// on, positions p0 .. p0 + PT, and the key blocks kb + 64 j, j < nblk: all of the
// tile's, or one segment of them.
struct QTile {
  static constexpr bool kRowTiles = true;
  int b, g, h0, heads, pad, p0, kb, nblk, tile, zero;  // zero: padded keys of the first block
  int split, all;                                      // the segment; blocks of the whole tile
  int lift;                                            // exponent of dS's factor
};
// A tile of keys k0 .. k0 + 128 of KV head g and the blocks of PT positions (from
// q0 on: earlier queries see none of these keys) x chunks of heads behind it.
struct KTile {
  static constexpr bool kRowTiles = false;
  int b, g, pad, k0, q0, per, nblk, tile, zero, split, lift;  // its blocks are split, split + splits, ...
};

// Key blocks that the rows before position `end` of a tile see.
__device__ __forceinline__ int row_blocks(int end, int pad, int S) {
  return (min(end, S) - 1 - (pad & ~7)) / kBlk + 1;
}

// Segments of seg blocks that a tile of `all` blocks is cut into.  A last one of a single
// block goes to the one before: the dq threads read the tile's dO and O before a
// segment's first scores, and only its second block's scores wait for them, so the last
// scores of a segment of one would give the tile's buffer back too early.
__host__ __device__ __forceinline__ int segments(int all, int seg) { return all <= seg + 1 ? 1 : (all + seg - 2) / seg; }

// fp16: the exponent of the factor of a unit's dS (attn_train_grad_max_kernel), 0 where there is no finite bound.  The
// loading thread takes it, its load beside that of the padding: at the start of an item, in the warps that use it,
// dq took 234 instead of 223 us for 2,048 x 192, 8 / 2 heads of 32.
struct GradExponent {
  const float2* part;
  float2 m;
  __device__ __forceinline__ GradExponent(const AttnTrainParams& p, int unit)
      : part(reinterpret_cast<const float2*>(p.grad_max) + (long long)unit * p.grad_parts), m(__ldg(part)) {}
  __device__ __forceinline__ int get(const AttnTrainParams& p) {
#pragma unroll 4
    for (int i = 1; i < p.grad_parts; ++i) {
      const float2 o = __ldg(part + i);
      m = make_float2(fmaxf(m.x, o.x), fmaxf(m.y, o.y));
    }
    const float c = 2.f * p.inv_keep * sqrtf(m.x * m.y);  // between 2^-47 and 2^56 unless 0 or infinite
    return c > 0.f && c < INFINITY ? 14 + 127 - (int)(__float_as_uint(c) >> 23) : 0;
  }
};

// The CTA's items: its own, then what it takes.  Taken no earlier than the loading
// thread needs it, a few blocks before the MMAs do.
template <class T, bool LIFT>
struct Items {
  static constexpr bool kRowTiles = T::kRowTiles;
  int claims = -1;
  bool more = true, ok = true;
  __device__ __forceinline__ int take(TcShared* sh, volatile int* abort, int* status) {
    const int i = claims < 0 ? (int)blockIdx.x : claim_item(sh, claims, abort, status, ok);
    ++claims;
    more = i >= 0;
    return i;
  }
  // False behind the last item, or (ok false) without an answer.
  __device__ __forceinline__ bool get(TcShared* sh, const AttnTrainParams& p, const Grid& gr, T& t) {
    const int i = take(sh, &sh->abort, p.status);
    if (i < 0) return false;
    const TcItem it = tc_item(gr, i, kRowTiles);
    const int bg = gr.by_parts(it.unit);
    struct {
      int b, g, part, tile, pad;
    } h;
    h.part = it.unit - bg * (gr.chunks > 1 && kRowTiles ? gr.chunks : gr.splits);
    h.b = gr.by_kv(bg);
    h.g = bg - h.b * p.Hkv;
    h.tile = it.tile;
    if constexpr (LIFT) {
      GradExponent e(p, bg);
      h.pad = p.pad_len ? __ldg(p.pad_len + h.b) : 0;
      t.lift = e.get(p);
    } else {
      h.pad = p.pad_len ? __ldg(p.pad_len + h.b) : 0;
      t.lift = 0;
    }
    t.b = h.b;
    t.g = h.g;
    t.pad = min(max(h.pad, 0), p.S);
    t.tile = h.tile;
    if constexpr (kRowTiles) {
      const int chunk = gr.chunks > 1 ? h.part : 0;
      t.split = gr.chunks > 1 ? 0 : h.part;
      t.h0 = h.g * p.R + chunk * p.HC;
      t.heads = min(p.HC, p.R - chunk * p.HC);
      t.p0 = t.pad + h.tile * p.PT128;
      t.all = t.p0 < p.S ? row_blocks(t.p0 + p.PT128, t.pad, p.S) : 0;
      t.kb = (t.pad & ~7) + t.split * gr.seg * kBlk;
      const int n = segments(t.all, gr.seg);
      t.nblk = t.split >= n ? 0 : t.split == n - 1 ? t.all - t.split * gr.seg : gr.seg;
      t.zero = t.split == 0 ? t.pad - t.kb : 0;
    } else {
      t.k0 = (t.pad & ~7) + h.tile * kRows;
      t.q0 = max(t.k0, t.pad);
      t.per = t.q0 < p.S ? p.by_pt64(p.S - t.q0 + p.PT64 - 1) : 0;
      t.split = h.part;
      t.nblk = gr.splits == 1 ? t.per * gr.chunks : max(0, t.per - h.part + gr.splits - 1) / gr.splits;
      t.zero = 0;
    }
    return true;
  }
};

// Whether the phase with this parity has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool warp_test(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_test(bar, parity));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status));
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

// Shared-memory matrix descriptors: the address is in the low word, so a thread
// that issues MMAs adds to 32 bits and joins the words in the instruction.
struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ Desc(const void* tile, uint32_t lbo, uint32_t sbo, uint32_t layout) {
    const uint64_t d = umma_smem_desc(smem_u32(tile), lbo, sbo, layout);
    lo = (uint32_t)d;
    hi = (uint32_t)(d >> 32);
  }
};
template <bool FIRST>
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\telect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(tmem_d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(FIRST ? 0 : 1)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\telect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

// Scores of one tile against one block: D[128 x 64] = A[128 x D] B[64 x D]^T; a_at and
// b_at move the descriptors to a tile buffer and a stage.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t tmem_d, const Desc& a, uint32_t a_at, const Desc& b,
                                             uint32_t b_at, uint32_t idesc) {
  const uint32_t al = a.lo + a_at, bl = b.lo + b_at;
  mma_ss<true>(tmem_d, al, a.hi, bl, b.hi, idesc);
#pragma unroll
  for (int kk = 1; kk < D / 16; ++kk) mma_ss<false>(tmem_d, al + 2 * kk, a.hi, bl + 2 * kk, b.hi, idesc);
}
// D[128 x D] += A[128 x 64] B[64 x D] with A in tensor memory: its first 32 columns
// in 16 columns of 32 bits, the others half_step columns further.
template <int D>
__device__ __forceinline__ void issue_weights(uint32_t tmem_d, uint32_t tmem_a, uint32_t half_step, const Desc& b,
                                              uint32_t b_at, uint32_t idesc, bool accumulate) {
  const uint32_t bl = b.lo + b_at;
#pragma unroll
  for (int kk = 0; kk < kBlk / 16; ++kk)
    mma_ts(tmem_d, tmem_a + (uint32_t)(kk >> 1) * half_step + (uint32_t)((kk & 1) * 8),
           bl + (uint32_t)(kk * 16 * TcShape<D>::ROWB >> 4), b.hi, idesc, kk > 0 ? 1u : (uint32_t)accumulate);
}

__device__ __forceinline__ void tc_init(TcShared* sh, int warps) {
  for (int i = 0; i < 2; ++i) {
    mbar_init(&sh->tile_full[i], 1);
    mbar_init(&sh->tile_empty[i], 1);
    mbar_init(&sh->s_full[i], 1);
    mbar_init(&sh->s_read[i], warps);
  }
  for (int i = 0; i < kMaxStages; ++i) {
    mbar_init(&sh->blk_full[i], 1);
    mbar_init(&sh->blk_empty[i], 1);
  }
  for (int i = 0; i < kItems; ++i) {
    mbar_init(&sh->item_full[i], 1);
    mbar_init(&sh->item_empty[i], warps);
  }
  for (int i = 0; i < 4; ++i) mbar_init(&sh->pair[i], 2);
  mbar_init(&sh->dp_full, 1);
  mbar_init(&sh->p_taken, 1);
  mbar_init(&sh->p_full, warps);
  mbar_init(&sh->ds_full, warps);
  mbar_init(&sh->w_done, 1);
  mbar_init(&sh->o_empty, warps);
  mbar_init(&sh->drain, 1);
  mbar_init(&sh->claimed, 1);
  sh->abort = 0;
  fence_mbar_init();
}

// The loading thread, the same for the three kernels: the tiles and blocks of the
// CTA's items in order, each into the next of TB tile buffers and STAGES stages,
// and each item's numbers into the ring that the element-wise warps read.
template <int TB, int STAGES, class T, bool LIFT, class Describe, class LoadTile, class LoadBlk>
__device__ __forceinline__ void load_all(TcShared* sh, const AttnTrainParams& p, const Grid& gr, Describe describe,
                                         LoadTile load_tile, LoadBlk load_blk) {
  volatile int* abort = &sh->abort;
  Items<T, LIFT> items;
  T t;
  int blocks = 0, tiles = 0, n = 0;
  bool ok = true, more = true;
  while (more) {
    more = items.get(sh, p, gr, t);
    if (!(ok = items.ok)) break;
    const int slot = n % kItems;
    if (!(ok = mbar_wait(&sh->item_empty[slot], ((n / kItems) & 1) ^ 1, abort, p.status))) break;
    if (more)
      describe(t, sh->item[slot]);
    else
      sh->item[slot].nblk = -1;
    mbar_arrive(&sh->item_full[slot]);
    ++n;
    if (!more || t.nblk == 0) continue;
    if (!(ok = mbar_wait(&sh->tile_empty[tiles % TB], ((tiles / TB) & 1) ^ 1, abort, p.status))) break;
    sh->tile_meta[tiles & 7] = make_int2(t.nblk, t.zero);
    load_tile(t, tiles % TB);
    ++tiles;
    for (int j = 0; j < t.nblk; ++j, ++blocks) {
      const int st = blocks % STAGES;
      if (!(ok = mbar_wait(&sh->blk_empty[st], ((blocks / STAGES) & 1) ^ 1, abort, p.status))) break;
      load_blk(t, j, st);
    }
    if (!ok) break;
  }
  // After an error the rest of the launch is taken and left, so that CTAs which wait in vain are few.
  if (!ok)
    while (items.more && items.ok) items.take(sh, nullptr, p.status);
  // Every copy must have landed before the CTA may end: after an error nobody else waits for them.
  for (int q = max(0, tiles - TB); q < tiles; ++q) mbar_wait(&sh->tile_full[q % TB], (q / TB) & 1, nullptr, nullptr);
  for (int q = max(0, blocks - STAGES); q < blocks; ++q)
    mbar_wait(&sh->blk_full[q % STAGES], (q / STAGES) & 1, nullptr, nullptr);
  if (ok && mbar_wait(&sh->tile_empty[tiles % TB], ((tiles / TB) & 1) ^ 1, abort, p.status)) {
    sh->tile_meta[tiles & 7] = make_int2(0, 0);
    mbar_arrive(&sh->tile_full[tiles % TB]);
  }
}

// The thread that issues the MMAs of the forward and dq kernels: SB score
// buffers, weights in columns of their own.
template <int SB, int TB, int STAGES, class Prepare, class Scores, class Weights>
__device__ __forceinline__ void issue_rows(TcShared* sh, int* status, Prepare prepare, Scores scores, Weights weights) {
  volatile int* abort = &sh->abort;
  int sblk = 0, stile = 0, sj = 0, sn = 0;  // next scores: block, tile, block within it, the tile's blocks
  bool ok = true, end = false;
  // Issues the next scores; without `wait` only if their operands are there.
  auto next_scores = [&](bool wait) {
    const int tb = stile % TB, st = sblk % STAGES;
    if (sj == 0) {
      if (!wait && !warp_test(&sh->tile_full[tb], (stile / TB) & 1)) return;
      if (!(ok = warp_wait(&sh->tile_full[tb], (stile / TB) & 1, abort, status))) return;
      sn = sh->tile_meta[stile & 7].x;
      if (sn == 0) {
        end = true;
        return;
      }
    }
    if (!wait && !warp_test(&sh->blk_full[st], (sblk / STAGES) & 1)) return;
    if (!(ok = warp_wait(&sh->blk_full[st], (sblk / STAGES) & 1, abort, status))) return;
    if (sj == 0) prepare(sh->tile_meta[stile & 7].y, st);
    tc_fence_after();
    scores(tb, st, sblk % SB);
    commit(&sh->s_full[sblk % SB]);
    ++sblk;
    if (++sj == sn) {
      commit(&sh->tile_empty[tb]);
      sj = 0;
      ++stile;
    }
  };
  int tiles = 0, j = 0, n = 0;  // the block whose weights come next: tile, block within it, the tile's blocks
  for (int blk = 0; ok; ++blk) {
    while (ok && !end && sblk <= blk) next_scores(true);
    if (!ok || sblk <= blk) break;
    if (SB > 1 && !end && sblk < blk + SB) next_scores(false);
    // The scores of this block being in registers, their buffer takes the next ones.
    if (!ok || !(ok = warp_wait(&sh->s_read[blk % SB], (blk / SB) & 1, abort, status))) break;
    if (!end && sblk == blk + SB) next_scores(false);
    if (!ok || !(ok = warp_wait(&sh->p_full, blk & 1, abort, status))) break;
    if (j == 0) {
      n = sh->tile_meta[tiles & 7].x;
      if (tiles > 0 && !(ok = warp_wait(&sh->o_empty, (tiles - 1) & 1, abort, status))) break;
    }
    tc_fence_after();
    weights(blk % STAGES, j > 0);
    commit(&sh->w_done);
    commit(&sh->blk_empty[blk % STAGES]);
    if (++j == n) {
      j = 0;
      ++tiles;
    }
  }
  commit(&sh->drain);
  warp_wait(&sh->drain, 0, nullptr, nullptr);
}

// The same for the dk, dv kernel: the two halves of a block in turn.  OVER: the weights
// lie over their scores, so the next scores wait until the product that reads them is
// done (P^T: p_taken, dS^T: the block's blk_empty).
template <int TB, int STAGES, bool OVER, class ScoresA, class ScoresB, class WeightsA, class WeightsB>
__device__ __forceinline__ void issue_keys(TcShared* sh, int* status, ScoresA scores_a, ScoresB scores_b,
                                           WeightsA weights_a, WeightsB weights_b) {
  volatile int* abort = &sh->abort;
  int a_blk = 0, a_tile = 0, a_j = 0, a_n = 0;  // next scores of the first half
  int b_blk = 0, b_tile = 0, b_j = 0;           // and of the second
  bool ok = true, end = false;
  auto next_a = [&](bool wait) {
    const int tb = a_tile % TB, st = a_blk % STAGES;
    if (a_j == 0) {
      if (!wait && !warp_test(&sh->tile_full[tb], (a_tile / TB) & 1)) return;
      if (!(ok = warp_wait(&sh->tile_full[tb], (a_tile / TB) & 1, abort, status))) return;
      a_n = sh->tile_meta[a_tile & 7].x;
      if (a_n == 0) {
        end = true;
        return;
      }
    }
    if (!wait && !warp_test(&sh->blk_full[st], (a_blk / STAGES) & 1)) return;
    if (!(ok = warp_wait(&sh->blk_full[st], (a_blk / STAGES) & 1, abort, status))) return;
    if (OVER && a_blk > 0 && !(ok = warp_wait(&sh->p_taken, (a_blk - 1) & 1, abort, status))) return;
    tc_fence_after();
    scores_a(tb, st);
    commit(&sh->s_full[0]);
    ++a_blk;
    if (++a_j == a_n) {
      a_j = 0;
      ++a_tile;
    }
  };
  auto next_b = [&]() {  // behind next_a of the same block, whose waits it shares
    if (OVER && b_blk > 0) {
      const int last = b_blk - 1;
      if (!(ok = warp_wait(&sh->blk_empty[last % STAGES], (last / STAGES) & 1, abort, status))) return;
      tc_fence_after();
    }
    scores_b(b_tile % TB, b_blk % STAGES);
    commit(&sh->dp_full);
    ++b_blk;
    if (++b_j == sh->tile_meta[b_tile & 7].x) {
      commit(&sh->tile_empty[b_tile % TB]);
      b_j = 0;
      ++b_tile;
    }
  };
  int tiles = 0, j = 0, n = 0;
  for (int blk = 0; ok; ++blk) {
    while (ok && !end && a_blk <= blk) next_a(true);
    if (!ok || a_blk <= blk) break;
    if (b_blk <= blk) next_b();
    if (!ok || !(ok = warp_wait(&sh->p_full, blk & 1, abort, status))) break;
    if (j == 0) {
      n = sh->tile_meta[tiles & 7].x;
      if (tiles > 0 && !(ok = warp_wait(&sh->o_empty, (tiles - 1) & 1, abort, status))) break;
    }
    tc_fence_after();
    weights_a(blk % STAGES, j > 0);
    if (OVER) commit(&sh->p_taken);
    if (!end) next_a(false);
    if (!ok || !(ok = warp_wait(&sh->ds_full, blk & 1, abort, status))) break;
    tc_fence_after();
    weights_b(blk % STAGES, j > 0);
    commit(&sh->blk_empty[blk % STAGES]);
    if (++j == n) {
      commit(&sh->w_done);
      j = 0;
      ++tiles;
    }
    if (b_blk < a_blk) next_b();
  }
  commit(&sh->drain);
  warp_wait(&sh->drain, 0, nullptr, nullptr);
}

// ---------------------------------------------------------------- scale of fp16 gradients
// |dS_j| = P_j |dP_j - delta| <= c = 2 / (1 - p) max|dO row| max|v row| (dP_j = m' dO . v_j, delta a mean of
// them), with the maxima over the rows of a sample and KV head behind its padding.  dS is scaled by the power of
// two that puts c into [2^14, 2^15): half of fp16's range is left for rounding, and what falls below its
// subnormals is below 2^-39 c.  Rows of squares' sums, NaN ignored; 2 D (Hq + Hkv) S bytes a sample to read,
// in parts of a unit that the readers join: 6 us for 1 x 5,003, 12 / 12 heads of 64, 34 for 96 x 768, 12 / 4 of 64,
// 42 for 2,048 x 192, 8 / 2 of 32.  The dq and dk, dv kernels take 3 to 8 % longer with it (the last two cases: 223 +
// 294 and 251 + 284 us, in bf16, which needs none of it, 208 + 288 and 244 + 272).
constexpr int kMaxGradParts = 32;

template <int D>
__global__ void __launch_bounds__(256) attn_train_grad_max_kernel(const __grid_constant__ AttnTrainParams p) {
  constexpr int NC = D / 8;  // threads of a row
  __shared__ uint32_t top[2][8];
  const int unit = blockIdx.x / p.grad_parts, part = blockIdx.x - unit * p.grad_parts;
  const int b = unit / p.Hkv, g = unit - b * p.Hkv;
  const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), p.S) : 0;
  const int per = (p.S - pad + p.grad_parts - 1) / p.grad_parts;
  const int first = min(pad + part * per, p.S), count = min(per, p.S - first);
  auto walk = [&](const void* base, long long ss, long long sh, int heads) {
    const uint16_t* at = static_cast<const uint16_t*>(base) + first * ss;
    // Row r is head r % heads of position r / heads; a turn's rows are stepped to without a division.  Several turns'
    // loads are in flight together.
    constexpr int kTurns = 4, kPerTurn = 256 / NC;
    const int c = threadIdx.x % NC, step = kPerTurn / heads, rest = kPerTurn % heads;
    int pos = threadIdx.x / NC / heads, head = threadIdx.x / NC % heads;
    float most = 0.f;
    for (long long r0 = 0; r0 < (long long)count * heads; r0 += kTurns * kPerTurn) {
      uint4 u[kTurns];
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        u[t] = pos < count ? *reinterpret_cast<const uint4*>(at + pos * ss + head * sh + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
        pos += step;
        head += rest;
        if (head >= heads) head -= heads, ++pos;
      }
#pragma unroll
      for (int t = 0; t < kTurns; ++t) {
        const uint32_t w[4] = {u[t].x, u[t].y, u[t].z, u[t].w};
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<false>::to_f2(w[e]);
          q = fmaf(f.x, f.x, fmaf(f.y, f.y, q));
        }
#pragma unroll
        for (int o = NC / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        most = fmaxf(most, q);
      }
    }
    return __reduce_max_sync(0xffffffffu, __float_as_uint(most));  // of floats from 0 up, by their bits
  };
  const uint32_t of_do = walk(static_cast<const uint16_t*>(p.dout) + b * p.do_sb + (long long)g * p.R * p.do_sh, p.do_ss,
                              p.do_sh, p.R);
  const uint32_t of_v = walk(static_cast<const uint16_t*>(p.v) + b * p.v_sb + g * p.v_sh, p.v_ss, p.v_sh, 1);
  if ((threadIdx.x & 31) == 0) {
    top[0][threadIdx.x >> 5] = of_do;
    top[1][threadIdx.x >> 5] = of_v;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, top[threadIdx.x][w]);
    p.grad_max[2 * (long long)blockIdx.x + threadIdx.x] = __uint_as_float(m);
  }
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The element-wise warps' side of the item ring.
struct ItemReader {
  TcShared* sh;
  volatile int* abort;
  int* status;
  int n = 0;
  __device__ __forceinline__ const Item* get(bool& ok) {  // the next item
    ok = warp_wait(&sh->item_full[n % kItems], (n / kItems) & 1, abort, status);
    return &sh->item[n % kItems];
  }
  __device__ __forceinline__ void next() {  // done with it (one lane of each warp says so)
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh->item_empty[n % kItems]);
    ++n;
  }
};

// Zeros the rows of a first block that lie before the padding's end (key block
// origin a multiple of 8), in both tensors of stage st.
template <int D>
__device__ __forceinline__ void zero_padded_keys(uint8_t* ring_a, uint8_t* ring_b, int st, int count) {
  using SH = TcShape<D>;
  if (count == 0) return;
  for (int e = threadIdx.x & 31; e < count * SH::NCH; e += 32) {
    *reinterpret_cast<uint4*>(ring_a + st * SH::BLK + e * 16) = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(ring_b + st * SH::BLK + e * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// ---------------------------------------------------------------- forward
constexpr int kFwdThreads = 192;  // a warpgroup of rows, the MMA warp, the loading warp

template <int D>
struct FwdSmem {
  using SH = TcShape<D>;
  static constexpr int OFF_K = 2 * SH::TILE;
  static constexpr int OFF_V = OFF_K + SH::STAGES * SH::BLK;
  static constexpr int OFF_SH = OFF_V + SH::STAGES * SH::BLK;
  static constexpr int NEED = OFF_SH + (int)sizeof(TcShared) + 1024;
  // Above a third of the SM's shared memory: two CTAs' 256 columns fill its tensor memory.
  static constexpr int BYTES = NEED > 78 * 1024 ? NEED : 78 * 1024;
  static_assert(kPerSm * (BYTES + 1024) <= 228 * 1024, "CTAs of an SM share its memory");
};

// CUT: tiles may be cut into segments (a form of its own, as for dq: 199 us instead of
// 187 for 2,048 x 192, 8 / 2 heads of 32, where none is cut).
template <int D, bool BF16, bool DROP, bool CUT>
__global__ void __launch_bounds__(kFwdThreads, kPerSm)
    attn_train_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                             const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnTrainParams p,
                             const __grid_constant__ Grid gr) {
  using SH = TcShape<D>;
  using SM = FwdSmem<D>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.S, PT = p.PT128, rows = PT * p.HC;

  if (tid == 0) tc_init(sh, 4);
  if (warp == 4) {
    tmem_alloc(&sh->tmem, kCols);
    tmem_relinquish();
  }
  zero_rows<SH::ROWB>(smem, 2, SH::TILE, rows, kRows, tid, kFwdThreads);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Columns: scores (one or two buffers), weights, O.
  const uint32_t t_s = sh->tmem, t_p = t_s + kFwdBufs * kBlk, t_o = t_p + kBlk / 2;
  volatile int* abort = &sh->abort;

  if (warp == 4) {
    const Desc qd(smem, 16, SH::SBO, SH::LAYOUT);
    const Desc kd(smem + SM::OFF_K, 16, SH::SBO, SH::LAYOUT);
    const Desc vd(smem + SM::OFF_V, SH::BLK, SH::SBO, SH::LAYOUT);
    const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
    issue_rows<kFwdBufs, 2, SH::STAGES>(
        sh, p.status,
        [&](int zero, int st) { zero_padded_keys<D>(smem + SM::OFF_K, smem + SM::OFF_V, st, zero); },
        [&](int tb, int st, int sb) {
          issue_scores<D>(t_s + (uint32_t)(sb * kBlk), qd, (uint32_t)(tb * (SH::TILE >> 4)), kd,
                          (uint32_t)(st * (SH::BLK >> 4)), id_s);
        },
        [&](int st, bool acc) { issue_weights<D>(t_o, t_p, 16, vd, (uint32_t)(st * (SH::BLK >> 4)), id_o, acc); });
  } else if (tid == 160) {
    load_all<2, SH::STAGES, QTile, false>(
        sh, p, gr,
        [&](const QTile& t, Item& it) {
          it.nblk = t.nblk, it.pad = t.pad, it.heads = t.heads, it.tile = t.tile;
          it.first = t.p0, it.origin = t.kb, it.split = t.split, it.per = t.all;
          it.row = ((long long)t.b * p.Hq + t.h0) * S;
          it.out = t.b * p.o_sb + t.h0 * p.o_sh;
        },
        [&](const QTile& t, int tb) {
          mbar_arrive_expect_tx(&sh->tile_full[tb], (uint32_t)(rows * SH::ROWB));
          tma_load_4d(smem + tb * SH::TILE, &tmQ, &sh->tile_full[tb], 0, t.h0, t.p0, t.b);
        },
        [&](const QTile& t, int j, int st) {
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * SH::BLK);
          tma_load_4d(smem + SM::OFF_K + st * SH::BLK, &tmK, &sh->blk_full[st], 0, t.g, t.kb + j * kBlk, t.b);
          tma_load_4d(smem + SM::OFF_V + st * SH::BLK, &tmV, &sh->blk_full[st], 0, t.g, t.kb + j * kBlk, t.b);
        });
  } else if (warp < 4) {
    const int r = tid, head = r % p.HC, rpos = r / p.HC;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t tp = t_p + lane_off, to = t_o + lane_off;
    const float c2 = p.scale * 1.4426950408889634f;
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    const uint32_t t2 = p.threshold * 0x10001u;
    DropKey key{};
    if constexpr (DROP) key = drop_key(p.rng, p.site);
    int blk = 0;
    bool ok = true;
    ItemReader items{sh, abort, p.status};
    // The finished tile: its O is read behind the next tile's first exponentials, when its last P V has long been done.
    struct {
      bool live, valid, partial;
      long long row;
      void* out;
      float m, l;
    } fin{};
    auto finish = [&]() {
      fin.live = false;
      uint32_t o[D];
#pragma unroll
      for (int c = 0; c < D; c += 32) tmem_ld32_async(to + c, *reinterpret_cast<uint32_t(*)[32]>(o + c));
#pragma unroll
      for (int c = 0; c < D; c += 32) tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(o + c));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->o_empty);
      if (CUT && fin.valid && fin.partial) {
        float* out = static_cast<float*>(fin.out);
#pragma unroll
        for (int c = 0; c < D; c += 4)
          *reinterpret_cast<uint4*>(out + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        *reinterpret_cast<float2*>(p.part_ml + 2 * fin.row) = make_float2(fin.m, fin.l);
      } else if (fin.valid) {
        const float inv = p.inv_keep / fin.l;
        uint16_t* out = static_cast<uint16_t*>(fin.out);
#pragma unroll
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + c) = pack8<BF16>(o + c, inv);
        p.lse[fin.row] = fin.m + log2f(fin.l);
      }
    };
    while (true) {
      const Item* it = items.get(ok);
      if (!ok) break;
      const int nblk = it->nblk, pad = it->pad, kb = it->origin, pos = it->first + rpos;
      if (nblk < 0) break;
      const bool mine = r < rows && head < it->heads, valid = mine && pos < S;
      const long long row = it->row + (long long)head * S + pos;
      uint16_t* out = static_cast<uint16_t*>(p.o) + it->out + head * p.o_sh;
      // This tile's share of the padded rows: zeros, each thread the row of its place.
      const int pz = it->tile * PT + rpos;
      const int split = CUT ? it->split : 0;
      const bool partial = CUT && segments(it->per, gr.seg) > 1;
      if (mine && pz < pad && split == 0) {
#pragma unroll
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + pz * p.o_ss + c) = make_uint4(0u, 0u, 0u, 0u);
        p.lse[row - pos + pz] = INFINITY;
      }
      items.next();
      const unsigned long long row_block = (unsigned long long)row * per_row;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nblk; ++j, ++blk) {
        const int sb = blk % kFwdBufs;
        if (!(ok = warp_wait(&sh->s_full[sb], (blk / kFwdBufs) & 1, abort, p.status))) break;
        tc_fence_after();
        const uint32_t ts = t_s + (uint32_t)(sb * kBlk) + lane_off;
        const int k0 = kb + j * kBlk;
        // Keys lo .. see - 1 of the block are the row's (a row without a query takes them all: it is not stored).
        const int see = valid ? pos - k0 + 1 : kBlk, lo = j == 0 ? pad - kb : 0;
        uint32_t s0[32], s1[32];
        tmem_ld32_async(ts, s0);
        tmem_ld32_async(ts + 32, s1);
        tmem_wait_ld(s0);
        tmem_wait_ld(s1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->s_read[sb]);
        if (lo > 0) {
#pragma unroll
          for (int i = 0; i < 7; ++i)
            if (i < lo) s0[i] = 0xff800000u;
        }
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
        const float mm = m == -INFINITY ? 0.f : m;
        const float2 c2v = make_float2(c2, c2), nm = make_float2(-mm, -mm);
        auto half = [&](uint32_t (&s)[32], int c) {  // leaves the packed weights in s[0 .. 16)
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int b8 = 0; b8 < 4; ++b8) {
            uint4 w8{};
            if constexpr (DROP) w8 = philox7(key, row_block + (unsigned)((k0 + 32 * c) / 8 + b8));
            const uint32_t words[4] = {w8.x, w8.y, w8.z, w8.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 8 * b8 + 2 * e;
              const float2 x = ffma2(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2v, nm);
              const float2 w = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              sum = fadd2(sum, w);
              s[i >> 1] = E::from_f2(w.x, w.y);
              // Dropped halves of the packed pair are cleared: a flag times 0xffff is its half's mask.
              if constexpr (DROP) s[i >> 1] &= ~(drop_flags(words[e], t2) * 0xffffu);
            }
          }
          l += sum.x + sum.y;
        };
        half(s0, 0);
        if (__any_sync(0xffffffffu, see > 32)) {
          half(s1, 1);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) s1[i] = 0u;
        }
        // The previous P V must be done before its weights are overwritten, or O scaled.
        if (blk > 0 && !(ok = warp_wait(&sh->w_done, (blk - 1) & 1, abort, p.status))) break;
        tc_fence_after();
        if (fin.live) finish();
        if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16_u(to + c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(to + c, o);
          }
        }
        tmem_st16(tp, *reinterpret_cast<uint32_t(*)[16]>(s0));
        tmem_st16(tp + 16, *reinterpret_cast<uint32_t(*)[16]>(s1));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      if (!ok) break;
      if (nblk > 0) {
        fin.live = true;
        fin.valid = valid;
        fin.partial = partial;
        fin.row = partial ? split * ((long long)p.B * p.Hq * S) + row : row;
        fin.out = partial ? static_cast<void*>(p.part + fin.row * D) : out + pos * p.o_ss;
        fin.m = m;
        fin.l = l;
      }
    }
    if (ok && fin.live && warp_wait(&sh->w_done, (blk - 1) & 1, abort, p.status)) {
      tc_fence_after();
      finish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(sh->tmem, kCols);
  }
}

// ---------------------------------------------------------------- dq
constexpr int kBwdThreads = 320;  // two warpgroups (half of a block's columns each), the MMA warp, the loading warp

template <int D, bool DQ>
struct BwdSmem {
  using SH = TcShape<D>;
  static constexpr int STAGES = DQ ? SH::DQ_STAGES : SH::STAGES;
  static constexpr int OFF_B = SH::BWD_TILES * SH::TILE;                // second tensor's tiles
  static constexpr int OFF_O = 2 * SH::BWD_TILES * SH::TILE;            // O's tiles (dq)
  static constexpr int OFF_C = OFF_O + (DQ ? SH::BWD_TILES * SH::TILE : 0);  // first ring
  static constexpr int OFF_E = OFF_C + STAGES * SH::BLK;                // second ring
  static constexpr int OFF_X = OFF_E + STAGES * SH::BLK;                // 4 KB of rows' scalars
  static constexpr int OFF_SH = OFF_X + 4096;
  static constexpr int NEED = OFF_SH + (int)sizeof(TcShared) + 1024;
  // Above a third of the SM's shared memory: two CTAs' 256 columns fill its tensor memory.
  static constexpr int BYTES = NEED > 78 * 1024 ? NEED : 78 * 1024;
  static_assert(kPerSm * (BYTES + 1024) <= 228 * 1024, "CTAs of an SM share its memory");
};

// CUT: tiles may be cut into segments (its registers spill: 250 us
// instead of 241 for 96 x 768, 12 / 4 heads of 64, where none is cut).
template <int D, bool BF16, bool DROP, bool CUT>
__global__ void __launch_bounds__(kBwdThreads, kPerSm)
    attn_train_dq_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                            const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ AttnTrainParams p, const __grid_constant__ Grid gr) {
  using SH = TcShape<D>;
  using SM = BwdSmem<D, true>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  float* xrow = reinterpret_cast<float*>(smem + SM::OFF_X);  // [2 items][2 halves][128] of delta
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.S, PT = p.PT128, rows = PT * p.HC;

  if (tid == 0) tc_init(sh, 8);
  if (warp == 8) {
    tmem_alloc(&sh->tmem, kCols);
    tmem_relinquish();
  }
  zero_rows<SH::ROWB>(smem, 2 * SH::BWD_TILES, SH::TILE, rows, kRows, tid, kBwdThreads);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Columns: S, dP, dS, dQ.
  const uint32_t t_s = sh->tmem, t_dp = t_s + kBlk, t_ds = t_dp + kBlk, t_dq = t_ds + kBlk / 2;
  volatile int* abort = &sh->abort;

  if (warp == 8) {
    const Desc qd(smem, 16, SH::SBO, SH::LAYOUT);
    const Desc dd(smem + SM::OFF_B, 16, SH::SBO, SH::LAYOUT);
    const Desc kd(smem + SM::OFF_C, 16, SH::SBO, SH::LAYOUT);
    const Desc vd(smem + SM::OFF_E, 16, SH::SBO, SH::LAYOUT);
    const Desc kt(smem + SM::OFF_C, SH::BLK, SH::SBO, SH::LAYOUT);
    const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
    issue_rows<1, SH::BWD_TILES, SH::DQ_STAGES>(
        sh, p.status,
        [&](int zero, int st) { zero_padded_keys<D>(smem + SM::OFF_C, smem + SM::OFF_E, st, zero); },
        [&](int tb, int st, int) {
          const uint32_t ta = (uint32_t)(tb * (SH::TILE >> 4)), sa = (uint32_t)(st * (SH::BLK >> 4));
          issue_scores<D>(t_s, qd, ta, kd, sa, id_s);
          issue_scores<D>(t_dp, dd, ta, vd, sa, id_s);
        },
        [&](int st, bool acc) { issue_weights<D>(t_dq, t_ds, 16, kt, (uint32_t)(st * (SH::BLK >> 4)), id_o, acc); });
  } else if (tid == 288) {
    load_all<SH::BWD_TILES, SH::DQ_STAGES, QTile, !BF16>(
        sh, p, gr,
        [&](const QTile& t, Item& it) {
          it.nblk = t.nblk, it.pad = t.pad, it.heads = t.heads, it.tile = t.tile;
          it.first = t.p0, it.origin = t.kb, it.split = t.split, it.per = t.all;
          it.row = ((long long)t.b * p.Hq + t.h0) * S;
          it.lift = t.lift;
          it.out = t.b * p.dq_sb + t.h0 * p.dq_sh;
        },
        [&](const QTile& t, int tb) {
          mbar_arrive_expect_tx(&sh->tile_full[tb], 3u * (uint32_t)(rows * SH::ROWB));
          tma_load_4d(smem + tb * SH::TILE, &tmQ, &sh->tile_full[tb], 0, t.h0, t.p0, t.b);
          tma_load_4d(smem + SM::OFF_B + tb * SH::TILE, &tmDO, &sh->tile_full[tb], 0, t.h0, t.p0, t.b);
          tma_load_4d(smem + SM::OFF_O + tb * SH::TILE, &tmO, &sh->tile_full[tb], 0, t.h0, t.p0, t.b);
        },
        [&](const QTile& t, int j, int st) {
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * SH::BLK);
          tma_load_4d(smem + SM::OFF_C + st * SH::BLK, &tmK, &sh->blk_full[st], 0, t.g, t.kb + j * kBlk, t.b);
          tma_load_4d(smem + SM::OFF_E + st * SH::BLK, &tmV, &sh->blk_full[st], 0, t.g, t.kb + j * kBlk, t.b);
        });
  } else if (warp < 8) {
    const int half = warp >> 2, wq = warp & 3, r = wq * 32 + lane;
    const int head = r % p.HC, rpos = r / p.HC;
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t ts = t_s + lane_off + 32 * half, tdp = t_dp + lane_off + 32 * half;
    const uint32_t tds = t_ds + lane_off + 16 * half;
    const float c2 = p.scale * 1.4426950408889634f;
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    DropKey key{};
    if constexpr (DROP) key = drop_key(p.rng, p.site);
    const long long all_rows = (long long)p.B * p.Hq * S;
    int blk = 0, done = 0;
    bool ok = true;
    ItemReader items{sh, abort, p.status};
    // The finished tile: its dQ is read behind the next tile's first weights.
    void* fin_out = nullptr;
    bool fin = false, fin_partial = false;
    auto finish = [&]() {
      fin = false;
#pragma unroll
      for (int c0 = 0; c0 < D / 2; c0 += 16) {
        uint32_t o[16];
        tmem_ld16_u(t_dq + lane_off + half * (D / 2) + c0, o);
        if (c0 + 16 == D / 2) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->o_empty);
        }
        const float out_scale = BF16 ? p.scale : *(volatile float*)&sh->out_scale[(done - 1) & 1][warp];
        if (CUT && fin_out && fin_partial) {
          float* out = static_cast<float*>(fin_out) + c0;
          if constexpr (!BF16)
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * out_scale);
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            *reinterpret_cast<uint4*>(out + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        } else if (fin_out) {
          uint16_t* out = static_cast<uint16_t*>(fin_out) + c0;
#pragma unroll
          for (int c = 0; c < 16; c += 8) *reinterpret_cast<uint4*>(out + c) = pack8<BF16>(o + c, out_scale);
        }
      }
    };
    while (true) {
      const Item* it = items.get(ok);
      if (!ok) break;
      const int nblk = it->nblk, pad = it->pad, kb = it->origin, pos = it->first + rpos;
      if (nblk < 0) break;
      const int lift = BF16 ? 0 : it->lift;
      const bool mine = r < rows && head < it->heads, valid = mine && pos < S;
      const long long row = it->row + (long long)head * S + pos;
      // A row with a single key (pos == pad) has no gradient: its P is taken as 0.
      const float ls = valid && pos != pad ? __ldg(p.lse + row) - (float)lift : INFINITY;
      uint16_t* out = static_cast<uint16_t*>(p.dq) + it->out + head * p.dq_sh + half * (D / 2);
      const int pz = it->tile * PT + rpos;
      const int split = CUT ? it->split : 0, all = CUT ? it->per : nblk;
      if (mine && pz < pad && split == 0) {
#pragma unroll
        for (int c = 0; c < D / 2; c += 8) *reinterpret_cast<uint4*>(out + pz * p.dq_ss + c) = make_uint4(0u, 0u, 0u, 0u);
      }
      items.next();
      out += pos * p.dq_ss;
      const unsigned long long row_block = (unsigned long long)row * per_row;
      // fp16: P, and so dS, is formed with dS's factor in its exponent (registers are short).
      if constexpr (!BF16) {
        *(volatile float*)&sh->inverse[warp] = power_of_two(-lift);
        *(volatile float*)&sh->out_scale[done & 1][warp] = p.scale * power_of_two(-lift);
      }
      float delta = 0.f;
      float* xr = xrow + (done & 1) * 2 * kRows;  // the other half may still be read for the previous item
      // The row's other half of delta comes from the warp of the other warpgroup, once for each item with blocks.
      // An mbarrier, not a barrier of the block: its wait has a limit, and a warp that has left after a failed wait
      // is not waited for without end.
      auto exchange = [&](float mine_half) {
        xr[half * kRows + r] = mine_half;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->pair[wq]);
        if (!warp_wait(&sh->pair[wq], done & 1, abort, p.status)) return false;
        delta = xr[r] + xr[kRows + r];
        return true;
      };
      if (nblk > 0 && all > 1) {
        // delta = O . dO: each of the row's two threads takes half of the columns.
        const int tb = done % SH::BWD_TILES;
        if (!(ok = warp_wait(&sh->tile_full[tb], (done / SH::BWD_TILES) & 1, abort, p.status))) break;
        float d = 0.f;
#pragma unroll
        for (int c = 0; c < SH::NCH / 2; ++c) {
          const uint32_t at = swz<SH::ROWB>(r, half * (SH::NCH / 2) + c) + tb * SH::TILE;
          const uint4 o = *reinterpret_cast<const uint4*>(smem + SM::OFF_O + at);
          const uint4 g = *reinterpret_cast<const uint4*>(smem + SM::OFF_B + at);
          const uint32_t a[4] = {o.x, o.y, o.z, o.w}, y[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 fa = E::to_f2(a[e]), fy = E::to_f2(y[e]);
            d = fmaf(fa.x, fy.x, fmaf(fa.y, fy.y, d));
          }
        }
        if (!(ok = exchange(d))) break;
        if (half == 0 && valid && split == 0) p.delta[row] = delta;
      }
      for (int j = 0; j < nblk; ++j, ++blk) {
        if (!(ok = warp_wait(&sh->s_full[0], blk & 1, abort, p.status))) break;
        tc_fence_after();
        const int k0 = kb + j * kBlk + 32 * half;
        const int see = valid ? pos - k0 + 1 : 32, lo = j == 0 && half == 0 ? pad - kb : 0;
        const bool any = __any_sync(0xffffffffu, valid && see > 0), edge = __any_sync(0xffffffffu, see < 32);
        uint32_t drop = 0;
        if constexpr (DROP) {
          if (any) {
            drop = drop_word(key, row_block + (unsigned)(k0 >> 3), p.threshold);
            if (p.words && valid) p.words[((k0 - (pad & ~7)) >> 5) * all_rows + row] = drop;
          }
        }
        // Columns c0 .. c0 + 16: P into w, dP (dropped, not yet scaled by 1 / (1 - p)) into d.
        auto chunk = [&](int c0, uint32_t (&w)[16], uint32_t (&d)[16]) {
          tmem_ld16_u(ts + c0, w);
          tmem_ld16_u(tdp + c0, d);
          if (c0 == 0 && lo > 0) {
#pragma unroll
            for (int c = 0; c < 7; ++c)
              if (c < lo) w[c] = 0xff800000u;
          }
          if (edge) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              if (c + c0 >= see) w[c] = 0xff800000u;
          }
          if constexpr (DROP) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              if (drop & drop_bit(c0 + c)) d[c] = 0u;
          }
          const float2 c2v = make_float2(c2, c2), nl = make_float2(-ls, -ls);
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            const float2 x = ffma2(make_float2(__uint_as_float(w[c]), __uint_as_float(w[c + 1])), c2v, nl);
            w[c] = __float_as_uint(ex2_approx(x.x));
            w[c + 1] = __float_as_uint(ex2_approx(x.y));
          }
        };
        if (all == 1) {
          // All keys of these rows are here: delta from the unrounded terms.
          float s = 0.f;
          if (any) {
#pragma unroll
            for (int c0 = 0; c0 < 32; c0 += 16) {
              uint32_t w[16], d[16];
              chunk(c0, w, d);
#pragma unroll
              for (int c = 0; c < 16; ++c) s = fmaf(__uint_as_float(w[c]), __uint_as_float(d[c]), s);
            }
          }
          if (!(ok = exchange(s * (BF16 ? p.inv_keep : p.inv_keep * *(volatile float*)&sh->inverse[warp])))) break;
          if (half == 0 && valid) p.delta[row] = delta;
          }
        uint32_t pk[16];
        if (any) {
          const float2 ik = make_float2(p.inv_keep, p.inv_keep), nd = make_float2(-delta, -delta);
#pragma unroll
          for (int c0 = 0; c0 < 32; c0 += 16) {
            uint32_t w[16], d[16];
            chunk(c0, w, d);
            if (c0 == 16) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh->s_read[0]);
            }
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const float2 g = make_float2(__uint_as_float(d[c]), __uint_as_float(d[c + 1]));
              const float2 x = fmul2(make_float2(__uint_as_float(w[c]), __uint_as_float(w[c + 1])),
                                     DROP ? ffma2(g, ik, nd) : fadd2(g, nd));
              pk[(c0 + c) >> 1] = E::from_f2(x.x, x.y);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) pk[c] = 0u;
          if (lane == 0) mbar_arrive(&sh->s_read[0]);
        }
        if (blk > 0 && !(ok = warp_wait(&sh->w_done, (blk - 1) & 1, abort, p.status))) break;
        tc_fence_after();
        if (fin) finish();
        tmem_st16(tds, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      if (!ok) break;
      if (nblk > 0) {
        ++done;
        fin = true;
        fin_partial = CUT && segments(all, gr.seg) > 1;
        fin_out = !valid ? nullptr
                  : fin_partial
                      ? static_cast<void*>(p.part + (split * all_rows + row) * D + half * (D / 2))
                      : out;
      }
    }
    if (ok && fin && warp_wait(&sh->w_done, (blk - 1) & 1, abort, p.status)) {
      tc_fence_after();
      finish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(sh->tmem, kCols);
  }
}

// ---------------------------------------------------------------- dk, dv
// WORDS: the drop flags come from the dq kernel (p.words).
template <int D, bool BF16, bool DROP, bool WORDS>
__global__ void __launch_bounds__(kBwdThreads, kPerSm)
    attn_train_dkv_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                             const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                             const __grid_constant__ AttnTrainParams p, const __grid_constant__ Grid gr) {
  using SH = TcShape<D>;
  using SM = BwdSmem<D, false>;
  using E = Elem<BF16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared* sh = reinterpret_cast<TcShared*>(smem + SM::OFF_SH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.S, PT = p.PT64, rows = PT * p.HC;

  if (tid == 0) tc_init(sh, 8);
  if (warp == 8) {
    tmem_alloc(&sh->tmem, kCols);
    tmem_relinquish();
  }
  zero_rows<SH::ROWB>(smem + SM::OFF_C, 2 * SH::STAGES, SH::BLK, rows, kBlk, tid, kBwdThreads);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Columns: S^T, dP^T, dV, dK, and P^T and dS^T behind them where there is room.
  constexpr bool OVER = 2 * kBlk + 2 * D + kBlk > (int)kCols;
  const uint32_t t_s = sh->tmem, t_dp = sh->tmem + 64, t_dv = sh->tmem + 128, t_dk = sh->tmem + 128 + D;
  const uint32_t t_p = OVER ? t_s : t_dk + D, t_ds = OVER ? t_dp : t_p + kBlk / 2, w_half = OVER ? 32 : 16;
  volatile int* abort = &sh->abort;

  if (warp == 8) {
    const Desc kd(smem, 16, SH::SBO, SH::LAYOUT);
    const Desc vd(smem + SM::OFF_B, 16, SH::SBO, SH::LAYOUT);
    const Desc qd(smem + SM::OFF_C, 16, SH::SBO, SH::LAYOUT);
    const Desc dd(smem + SM::OFF_E, 16, SH::SBO, SH::LAYOUT);
    const Desc qt(smem + SM::OFF_C, SH::BLK, SH::SBO, SH::LAYOUT);
    const Desc dt(smem + SM::OFF_E, SH::BLK, SH::SBO, SH::LAYOUT);
    const uint32_t id_s = umma_idesc_f16(BF16, kRows, kBlk, 0, 0), id_o = umma_idesc_f16(BF16, kRows, D, 0, 1);
    auto tile_at = [](int tb) { return (uint32_t)(tb * (SH::TILE >> 4)); };
    auto blk_at = [](int st) { return (uint32_t)(st * (SH::BLK >> 4)); };
    issue_keys<SH::BWD_TILES, SH::STAGES, OVER>(
        sh, p.status,
        [&](int tb, int st) { issue_scores<D>(t_s, kd, tile_at(tb), qd, blk_at(st), id_s); },
        [&](int tb, int st) { issue_scores<D>(t_dp, vd, tile_at(tb), dd, blk_at(st), id_s); },
        [&](int st, bool acc) { issue_weights<D>(t_dv, t_p, w_half, dt, blk_at(st), id_o, acc); },
        [&](int st, bool acc) { issue_weights<D>(t_dk, t_ds, w_half, qt, blk_at(st), id_o, acc); });
  } else if (tid == 288) {
    load_all<SH::BWD_TILES, SH::STAGES, KTile, !BF16>(
        sh, p, gr,
        [&](const KTile& t, Item& it) {
          it.nblk = t.nblk, it.pad = t.pad, it.tile = t.tile;
          it.first = t.q0, it.origin = t.k0, it.per = t.per, it.split = t.split;
          it.row = ((long long)t.b * p.Hq + t.g * p.R) * S;
          it.lift = t.lift;
          it.out = t.b * p.dv_sb + t.g * p.dv_sh;
          it.out2 = t.b * p.dk_sb + t.g * p.dk_sh;
          it.part = (((long long)t.split * 2 * p.B + t.b) * p.Hkv + t.g) * S;
        },
        [&](const KTile& t, int tb) {
          mbar_arrive_expect_tx(&sh->tile_full[tb], 2u * SH::TILE);
          tma_load_4d(smem + tb * SH::TILE, &tmK, &sh->tile_full[tb], 0, t.g, t.k0, t.b);
          tma_load_4d(smem + SM::OFF_B + tb * SH::TILE, &tmV, &sh->tile_full[tb], 0, t.g, t.k0, t.b);
        },
        [&](const KTile& t, int j, int st) {
          const int c = gr.chunks > 1 ? j / t.per : 0, h0 = c * p.HC;
          const int q0 = t.q0 + (t.split + j * gr.splits - c * t.per) * PT;
          mbar_arrive_expect_tx(&sh->blk_full[st], 2u * (uint32_t)(rows * SH::ROWB));
          tma_load_5d(smem + SM::OFF_C + st * SH::BLK, &tmQ, &sh->blk_full[st], 0, h0, t.g, q0, t.b);
          tma_load_5d(smem + SM::OFF_E + st * SH::BLK, &tmDO, &sh->blk_full[st], 0, h0, t.g, q0, t.b);
        });
  } else if (warp < 8) {
    const int half = warp >> 2, wq = warp & 3;
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t ts = t_s + lane_off + 32 * half, tdp = t_dp + lane_off + 32 * half;
    const uint32_t tp = t_p + lane_off + w_half * half, tds = t_ds + lane_off + w_half * half;
    const float c2 = p.scale * 1.4426950408889634f;
    const float2 c2v = make_float2(c2, c2);
    constexpr float kLift = BF16 ? 0.f : 15.f;           // of P, as a power of two
    constexpr float kLower = BF16 ? 1.f : 1.f / 32768.f;  // and out again
    DropKey key{};
    const unsigned per_row = (unsigned)(S + 7) >> 3;
    if constexpr (DROP && !WORDS) key = drop_key(p.rng, p.site);
    const long long all_rows = (long long)p.B * p.Hq * S;
    // Scalars of the warp's 32 columns (query rows): lane l fetches those of column l; 4-byte arrays read in fours.
    float* x_nl = reinterpret_cast<float*>(smem + SM::OFF_X) + warp * 32;                 // -lse
    float* x_nd = reinterpret_cast<float*>(smem + SM::OFF_X + 1024) + warp * 32;          // -delta
    int* x_pos = reinterpret_cast<int*>(smem + SM::OFF_X + 2048) + warp * 32;
    const int col = 32 * half + lane, chead = col % p.HC, cpos = col / p.HC;
    const int first_pos = 32 * half / p.HC, last_pos = min(32 * half + 31, rows - 1) / p.HC;
    int blk = 0, done = 0;
    bool ok = true;
    ItemReader items{sh, abort, p.status};
    // The finished tile: dv (first warpgroup) or dk (second) is read when the next tile's first scores are there.
    uint16_t* fin_out = nullptr;
    float* fin_part = nullptr;
    bool fin = false;
    float fin_inv = 1.f;  // fp16: takes dS's factor out
    auto finish = [&]() {
      fin = false;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32_async((half ? t_dk : t_dv) + lane_off + c, o);
        tmem_wait_ld(o);
        if (c + 32 == D) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->o_empty);
        }
        if (fin_part) {
          if constexpr (!BF16)
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * (half ? fin_inv : kLower));
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(fin_part + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else if (fin_out)
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(fin_out + c + e) = pack8<BF16>(o + e, half ? (BF16 ? p.scale : p.scale * fin_inv) : p.inv_keep * kLower);
      }
    };
    while (true) {
      const Item* it = items.get(ok);
      if (!ok) break;
      const int nblk = it->nblk, pad = it->pad, per = it->per;
      const int first = it->first + it->split * PT, step = gr.splits * PT;
      if (nblk < 0) break;
      const int lift = BF16 ? 0 : it->lift;
      const float factor = power_of_two(lift) * kLower;  // dS has P's lift as well
      const float2 ik = make_float2(p.inv_keep * factor, p.inv_keep * factor);
      const int key0 = it->origin + wq * 32, kk = key0 + lane;  // the warp's keys, the thread's
      const int it_tile = it->tile;
      const long long row_at = it->row;
      uint16_t* out = half ? static_cast<uint16_t*>(p.dk) + it->out2 : static_cast<uint16_t*>(p.dv) + it->out;
      const long long out_ss = half ? p.dk_ss : p.dv_ss;
      const int pz = it_tile * kRows + wq * 32 + lane;
      if (pz < pad && it->split == 0) {
#pragma unroll
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + pz * out_ss + c) = make_uint4(0u, 0u, 0u, 0u);
      }
      float* part = gr.splits > 1 ? p.part + (it->part + (half ? (long long)p.B * p.Hkv * S : 0)) * D : nullptr;
      items.next();
      // Position and row of the thread's column in the block whose scalars are fetched next, and those scalars.
      int npos = first + cpos;
      long long nrow = row_at + (long long)chead * S + npos;
      float nl = -INFINITY, nd = 0.f;
      uint32_t nw = 0;
      const uint32_t* words = nullptr;
      if constexpr (WORDS) words = p.words + (it_tile * 4 + wq) * all_rows;
      auto fetch = [&](int j) {
        if (gr.chunks > 1 && j > 0 && j % per == 0) {  // the next chunk of heads, from the first position again
          npos = first + cpos;
          nrow = row_at + (long long)(j / per * p.HC + chead) * S + npos;
        }
        const bool there = j < nblk && col < rows && npos < S && (gr.chunks == 1 || j / per * p.HC + chead < p.R);
        nl = there ? kLift - __ldg(p.lse + nrow) : -INFINITY;
        nd = there ? -__ldg(p.delta + nrow) * factor : 0.f;
        if constexpr (WORDS) nw = there && npos >= key0 ? __ldg(words + nrow) : 0u;  // written where a key is seen
      };
      fetch(0);
      for (int j = 0; j < nblk; ++j, ++blk) {
        const int pos = npos, q0 = pos - cpos;
        const long long row = nrow;
        // The warp's last position against its first key: nothing to do where every query comes before every key
        // (or where the warp has no query or no key).
        const bool any = q0 + last_pos >= key0 && key0 < S && q0 + first_pos < S;
        uint32_t drop = nw;
        if constexpr (DROP && !WORDS) {
          if (any) drop = drop_word(key, (unsigned long long)row * per_row + (unsigned)(key0 >> 3), p.threshold);
        }
        // From the flags of a column's 32 keys to those of the thread's key in 32 columns.
        if constexpr (DROP) drop = __shfl_sync(0xffffffffu, warp_transpose(drop, lane), drop_place(lane));
        __syncwarp();
        x_nl[lane] = nl;
        x_nd[lane] = nd;
        x_pos[lane] = pos;
        __syncwarp();
        // The next block's scalars: on their way while this one is worked on.
        npos += step;
        nrow += step;
        fetch(j + 1);
        if (!(ok = warp_wait(&sh->s_full[0], blk & 1, abort, p.status))) break;
        tc_fence_after();
        if (fin) {
          if (!(ok = warp_wait(&sh->w_done, (done - 1) & 1, abort, p.status))) break;
          tc_fence_after();
          finish();
        }
        uint32_t s[32];
        if (any) {
          tmem_ld32_async(ts, s);
          tmem_wait_ld(s);
          // Only blocks on the diagonal hold queries before a key.
          if (q0 < key0 + 31) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (kk > x_pos[c]) s[c] = 0xff800000u;
          }
#pragma unroll
          for (int c0 = 0; c0 < 32; c0 += 16) {
            uint32_t pw[8];
#pragma unroll
            for (int c4 = c0; c4 < c0 + 16; c4 += 4) {
              const float4 nl4 = *reinterpret_cast<const float4*>(x_nl + c4);
#pragma unroll
              for (int c = c4; c < c4 + 4; c += 2) {
                const float2 x = ffma2(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2v,
                                       c == c4 ? make_float2(nl4.x, nl4.y) : make_float2(nl4.z, nl4.w));
                const float w0 = ex2_approx(x.x), w1 = ex2_approx(x.y);
                s[c] = __float_as_uint(w0);
                s[c + 1] = __float_as_uint(w1);
                if constexpr (DROP)
                  pw[(c - c0) >> 1] = E::from_f2(drop & 1u << c ? 0.f : w0, drop & 2u << c ? 0.f : w1);
                else
                  pw[(c - c0) >> 1] = E::from_f2(w0, w1);
              }
            }
            tmem_st8(tp + (c0 >> 1), pw);
          }
        } else {
          uint32_t z[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) z[c] = 0u;
          tmem_st8(tp, z);
          tmem_st8(tp + 8, z);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
        if (!(ok = warp_wait(&sh->dp_full, blk & 1, abort, p.status))) break;
        tc_fence_after();
        if (any) {
          // The row with a single key (position pad) has no dS.
          if (q0 == pad) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (x_pos[c] == pad) s[c] = 0u;
          }
#pragma unroll
          for (int c0 = 0; c0 < 32; c0 += 16) {
            uint32_t dp[16];
            tmem_ld16_u(tdp + c0, dp);
#pragma unroll
            for (int c4 = 0; c4 < 16; c4 += 4) {
              const float4 nd4 = *reinterpret_cast<const float4*>(x_nd + c0 + c4);
#pragma unroll
              for (int c = c4; c < c4 + 4; c += 2) {
                const float2 md = c == c4 ? make_float2(nd4.x, nd4.y) : make_float2(nd4.z, nd4.w);
                float2 d = make_float2(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1]));
                if constexpr (DROP)
                  d = ffma2(make_float2(drop & 1u << (c0 + c) ? 0.f : d.x, drop & 2u << (c0 + c) ? 0.f : d.y), ik, md);
                else
                  d = BF16 ? fadd2(d, md) : ffma2(d, ik, md);
                d = fmul2(make_float2(__uint_as_float(s[c0 + c]), __uint_as_float(s[c0 + c + 1])), d);
                s[(c0 + c) >> 1] = E::from_f2(d.x, d.y);
              }
            }
          }
          tmem_st16(tds, *reinterpret_cast<uint32_t(*)[16]>(s));
        } else {
          uint32_t z[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) z[c] = 0u;
          tmem_st16(tds, z);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ds_full);
      }
      if (!ok) break;
      if (nblk > 0) {
        ++done;
        fin = true;
        if constexpr (!BF16) fin_inv = power_of_two(-lift);
        const bool kept = kk >= pad && kk < S;
        fin_out = kept ? out + kk * out_ss : nullptr;
        fin_part = kept && part ? part + (long long)kk * D : nullptr;
      }
    }
    if (ok && fin && warp_wait(&sh->w_done, (done - 1) & 1, abort, p.status)) {
      tc_fence_after();
      finish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(sh->tmem, kCols);
  }
}

// Adds the splits' sums of dk and dv in order: eight columns of a row a thread.  A
// tile has sums from as many splits as it has blocks, at most all.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attn_train_sum_kernel(const __grid_constant__ AttnTrainParams p, int splits) {
  constexpr int NC = D / 8;
  const long long rows = (long long)p.B * p.Hkv * p.S, total = rows * 2 * NC;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int c = (int)(i % NC) * 8, which = (int)(i / NC % 2);
    const long long row = i / (2 * NC);
    const int pos = (int)(row % p.S);
    const long long bg = row / p.S;
    const int g = (int)(bg % p.Hkv), b = (int)(bg / p.Hkv), pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), p.S) : 0;
    if (pos < pad) continue;
    const int k0 = (pad & ~7) + (pos - (pad & ~7)) / kRows * kRows;
    const int n = min(splits, (p.S - max(k0, pad) + p.PT64 - 1) / p.PT64);
    const float* src = p.part + (which * rows + row) * D + c;
    uint32_t s[8];
    float acc[8] = {};
    for (int q = 0; q < n; ++q, src += 2 * rows * D) {
      const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
      acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
      acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = __float_as_uint(acc[e]);
    uint16_t* dst = which ? static_cast<uint16_t*>(p.dk) + b * p.dk_sb + (long long)pos * p.dk_ss + g * p.dk_sh
                          : static_cast<uint16_t*>(p.dv) + b * p.dv_sb + (long long)pos * p.dv_ss + g * p.dv_sh;
    *reinterpret_cast<uint4*>(dst + c) = pack8<BF16>(s, which ? p.scale : p.inv_keep);
  }
}

// Joins the segments of the tiles of rows that were cut, eight columns of a row a
// thread, in order.  Forward: O and the sums l to the largest of the segments'
// references m, then O / l and lse.  dq: the sum.
template <int D, bool BF16, bool FWD>
__global__ void __launch_bounds__(256) attn_train_join_kernel(const __grid_constant__ AttnTrainParams p, int seg) {
  constexpr int NC = D / 8;
  const long long rows = (long long)p.B * p.Hq * p.S, total = rows * NC;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int c = (int)(i % NC) * 8;
    const long long row = i / NC, bh = row / p.S;
    const int pos = (int)(row - bh * p.S), b = (int)(bh / p.Hq), h = (int)(bh - (long long)b * p.Hq);
    const int pad = p.pad_len ? min(max(__ldg(p.pad_len + b), 0), p.S) : 0;
    if (pos < pad) continue;
    const int all = row_blocks(pad + ((pos - pad) / p.PT128 + 1) * p.PT128, pad, p.S);
    const int n = segments(all, seg);
    if (n == 1) continue;
    float top = -INFINITY, l = 0.f;
    if constexpr (FWD)
      for (int q = 0; q < n; ++q) top = fmaxf(top, p.part_ml[2 * (q * rows + row)]);
    float acc[8] = {};
    const float* src = p.part + row * D + c;
    for (int q = 0; q < n; ++q, src += rows * D) {
      const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      float f = 1.f;
      if constexpr (FWD) {
        // A segment without a key of this row (all behind it) has m = -inf and zeros.
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (q * rows + row));
        f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
        l = fmaf(ml.y, f, l);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(v[e], f, acc[e]);
    }
    uint32_t s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = __float_as_uint(acc[e]);
    if constexpr (FWD) {
      uint16_t* out = static_cast<uint16_t*>(p.o) + b * p.o_sb + (long long)pos * p.o_ss + h * p.o_sh;
      *reinterpret_cast<uint4*>(out + c) = pack8<BF16>(s, p.inv_keep / l);
      if (c == 0) p.lse[row] = top + log2f(l);
    } else {
      uint16_t* out = static_cast<uint16_t*>(p.dq) + b * p.dq_sb + (long long)pos * p.dq_ss + h * p.dq_sh;
      *reinterpret_cast<uint4*>(out + c) = pack8<BF16>(s, BF16 ? p.scale : 1.f);  // fp16: scaled with the factor taken out
    }
  }
}

int row_blocks_most(int S) { return (S + 7 + kBlk - 1) / kBlk; }  // of any tile, whatever the padding
Grid make_grid(const AttnTrainParams& p, int units, int tiles, int parts, int splits, int seg) {
  return Grid{units * parts, tiles, units * parts * tiles, (p.R + p.HC - 1) / p.HC, splits, seg,
              FastDiv((uint32_t)tiles), FastDiv((uint32_t)parts), FastDiv((uint32_t)p.Hkv)};
}
Grid grid_rows(const AttnTrainParams& p, int num_sms) {
  const int chunks = (p.R + p.HC - 1) / p.HC, splits = attn_train_row_splits(p.B, p.S, p.Hkv, p.R, num_sms);
  return make_grid(p, p.B * p.Hkv, (p.S + p.PT128 - 1) / p.PT128, chunks > 1 ? chunks : splits, splits,
                   (row_blocks_most(p.S) + splits - 1) / splits);
}
Grid grid_keys(const AttnTrainParams& p, int splits) {
  return make_grid(p, p.B * p.Hkv, (p.S + kRows - 1) / kRows, splits, splits, 0);
}
template <int D, bool BF16, bool FWD>
cudaError_t join(const AttnTrainParams& p, const Grid& gr, int num_sms, cudaStream_t st) {
  if (gr.splits == 1) return cudaSuccess;
  const long long blocks = ((long long)p.B * p.Hq * p.S * (D / 8) + 255) / 256;
  attn_train_join_kernel<D, BF16, FWD><<<(unsigned)(blocks < num_sms * 16 ? blocks : num_sms * 16), 256, 0, st>>>(p, gr.seg);
  return cudaGetLastError();
}
template <int D, bool BF16, bool DROP>
cudaError_t run_fwd(const AttnTrainParams& p, const AttnTrainMaps& m, int num_sms, cudaStream_t st) {
  const Grid gr = grid_rows(p, num_sms);
  auto kern = gr.splits > 1 ? attn_train_fwd_tc_kernel<D, BF16, DROP, true> : attn_train_fwd_tc_kernel<D, BF16, DROP, false>;
  cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kern), FwdSmem<D>::BYTES);
  if (e != cudaSuccess) return e;
  kern<<<(unsigned)gr.items, kFwdThreads, FwdSmem<D>::BYTES, st>>>(m.q_tile, m.k_blk, m.v_blk, p, gr);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return join<D, BF16, true>(p, gr, num_sms, st);
}
template <int D, bool BF16, bool DROP>
cudaError_t run_bwd(const AttnTrainParams& p, const AttnTrainMaps& m, int num_sms, cudaStream_t st) {
  const Grid gq = grid_rows(p, num_sms);
  auto kq = gq.splits > 1 ? attn_train_dq_tc_kernel<D, BF16, DROP, true> : attn_train_dq_tc_kernel<D, BF16, DROP, false>;
  auto kk = DROP && p.words ? attn_train_dkv_tc_kernel<D, BF16, DROP, DROP> : attn_train_dkv_tc_kernel<D, BF16, DROP, false>;
  cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kq), BwdSmem<D, true>::BYTES);
  if (e != cudaSuccess) return e;
  if ((e = smem_limit_once(reinterpret_cast<const void*>(kk), BwdSmem<D, false>::BYTES)) != cudaSuccess) return e;
  const int splits = attn_train_splits(p.B, p.S, p.Hkv, p.R, num_sms);
  const Grid gk = grid_keys(p, splits);
  if constexpr (!BF16) {
    attn_train_grad_max_kernel<D><<<(unsigned)(p.B * p.Hkv * p.grad_parts), 256, 0, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  kq<<<(unsigned)gq.items, kBwdThreads, BwdSmem<D, true>::BYTES, st>>>(m.q_tile, m.do_tile, m.o_tile, m.k_blk,
                                                                              m.v_blk, p, gq);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = join<D, BF16, false>(p, gq, num_sms, st)) != cudaSuccess) return e;
  kk<<<(unsigned)gk.items, kBwdThreads, BwdSmem<D, false>::BYTES, st>>>(m.k_tile, m.v_tile, m.q_blk, m.do_blk, p, gk);
  if ((e = cudaGetLastError()) != cudaSuccess || splits == 1) return e;
  const long long blocks = ((long long)p.B * p.Hkv * p.S * 2 * (D / 8) + 255) / 256;
  attn_train_sum_kernel<D, BF16><<<(unsigned)(blocks < num_sms * 16 ? blocks : num_sms * 16), 256, 0, st>>>(p, splits);
  return cudaGetLastError();
}

}  // namespace

// CTAs that share the query rows behind one tile of keys.  The first tile of a
// causal unit has twice the average's rows, so that a few tiles are cut until there
// are about two items for each CTA of the GPU, with eight blocks or more for each
// (B 2, S 4000, 8 / 2 heads of 32, 128 tiles for 296 CTAs: 166 us cut in two, 120 us
// in three, 97 us in four and in six; B 7, S 1305, 16 / 4 heads of 32, 308 tiles: 130 us
// whole, 76 in two and 5 for the sum; B 64, S 192, twelve blocks in the longest of 256
// tiles: 24 us whole, 29 us with the sum cut in two).
int attn_train_splits(int B, int S, int Hkv, int R, int num_sms) {
  if (R > 64) return 1;  // chunks of heads: not split
  const long long items = (long long)B * Hkv * ((S + kRows - 1) / kRows);
  const int pt = kBlk / R, blocks = (S + pt - 1) / pt;
  long long n = (2LL * kPerSm * num_sms + items / 2) / items;
  if (n > blocks / 8) n = blocks / 8;
  return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}

// Segments of the longest tile of query rows' key blocks, each its own item: the same
// rule for the walk over keys, but rounded down, as there are two joins to pay for
// (rounded to the nearest, forward and dq: 3 x 1800, 8 / 2 heads of 32 43 + 47 -> 42 + 45 us
// with the forward join, but 2 x 2000, 12 heads of 64 35 + 37 -> 45 + 43, 1 x 1100, 40 heads
// of 64 22 + 24 -> 33 + 30, 1 x 4096, 12 heads of 64 95 + 110 -> 96 + 112).
int attn_train_row_splits(int B, int S, int Hkv, int R, int num_sms) {
  if (R > 64) return 1;
  const int pt = kRows / R;
  const long long items = (long long)B * Hkv * ((S + pt - 1) / pt);
  long long n = 2LL * kPerSm * num_sms / items;
  const int blocks = row_blocks_most(S);
  if (n > blocks / 8) n = blocks / 8;
  return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}

// Words of drop flags that the dq kernel hands to the dk, dv kernel, 0 where both
// generate them.
long long attn_train_words(int B, int S, int Hq, int D) {
  if (S > kWordsPerDim * D) return 0;
  return (long long)B * Hq * S * ((S + kBlk - 1) / kBlk * 2);
}

// Blocks that share the rows of a sample and KV head in attn_train_grad_max_kernel: about
// eight 16-byte loads a thread.
int attn_train_grad_parts(int S, int R, int D) {
  const long long n = (long long)S * (R + 1) * (D / 8) / 2048;
  return (int)(n < 1 ? 1 : n > kMaxGradParts ? kMaxGradParts : n);
}

cudaError_t launch_attn_train_fwd_sm100(const AttnTrainParams& p, const AttnTrainMaps& m, int D, bool bf16,
                                        int num_sms, cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? run_fwd<32, true, true>(p, m, num_sms, st) : run_fwd<32, true, false>(p, m, num_sms, st))
                : (drop ? run_fwd<32, false, true>(p, m, num_sms, st) : run_fwd<32, false, false>(p, m, num_sms, st));
  return bf16 ? (drop ? run_fwd<64, true, true>(p, m, num_sms, st) : run_fwd<64, true, false>(p, m, num_sms, st))
              : (drop ? run_fwd<64, false, true>(p, m, num_sms, st) : run_fwd<64, false, false>(p, m, num_sms, st));
}

cudaError_t launch_attn_train_bwd_sm100(const AttnTrainParams& p, const AttnTrainMaps& m, int D, bool bf16,
                                        int num_sms, cudaStream_t st) {
  const bool drop = p.threshold != 0;
  if (D == 32)
    return bf16 ? (drop ? run_bwd<32, true, true>(p, m, num_sms, st) : run_bwd<32, true, false>(p, m, num_sms, st))
                : (drop ? run_bwd<32, false, true>(p, m, num_sms, st) : run_bwd<32, false, false>(p, m, num_sms, st));
  return bf16 ? (drop ? run_bwd<64, true, true>(p, m, num_sms, st) : run_bwd<64, true, false>(p, m, num_sms, st))
              : (drop ? run_bwd<64, false, true>(p, m, num_sms, st) : run_bwd<64, false, false>(p, m, num_sms, st));
}

}  // namespace dtk
