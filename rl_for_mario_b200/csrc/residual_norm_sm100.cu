// Residual add with the norms before and after it, a gate and dropout, and its
// gradient: what stands between two blocks' products in training, one pass.
//
//   u = x * r_post * w_post   r_post = rsqrt(mean(x^2) + eps)   (u = x without a post norm)
//   v = m u / (1 - p)         m the dropout mask (philox.cuh)
//   h = residual + alpha * g * v
//   n = h * r_pre * w_pre     r_pre = rsqrt(mean(h^2) + eps)
//
// Backward, from dh (the gradient that reaches h past this op) and dn, with
// h^ = h r_pre and x^ = x r_post:
//   t  = dn * w_pre,  e = dh + r_pre t,  c = mean(t h^)
//   D  = e - r_pre c h^                      the gradient of h: d(residual) = D
//   dg = alpha v D (summed over the rows that share a gate),  du = m alpha g D / (1 - p)
//   s  = du * w_post, d(x) = r_post (s - x^ c')     (d(x) = du without a post norm)
//   dw_pre = sum over rows of dn h^,  dw_post = sum over rows of du x^
// c' = mean(s x^) looks as if it had to wait for c, but s x^ = (alpha g v) D, so
//   c' = mean(alpha g v e) - r_pre c mean(alpha g v h^),
// and one sum over the row gives all three means.
// h is formed again from x and residual in fp32 instead of being read back, so the
// gradient does not see the rounding of the stored h.  With a post norm or a gate x is
// needed anyway and the bytes are the same; without either it is one tensor more to read.
//
// Everything between the loads and the stores is fp32; each output is rounded
// once, and n is the norm of the unrounded h.
//
// Bound by HBM.  A row is held by one or more warps (WPR), so it is read once and
// its sums are a shuffle tree plus (WPR > 1) one named barrier; the next rows' loads
// are issued before this row's sums, so that they are in flight behind the barriers.
// The sums over rows of the backward pass stay in registers (a thread owns its columns
// for every row that it meets); one block of up to 512 threads on each SM writes one
// partial row of them and a second kernel adds the partial rows in a fixed order: no
// atomics, the same bits every run.  96 x 768 rows of 768, bf16, both norms and a gate:
// 88 us forward (453 MB, 5.1 TB/s), 132 us backward (680 MB, 5.2 TB/s) and 3 us for the
// sums; what is left to the 6.5 TB/s of a copy goes to the two (one) row sums that
// every row waits for, with 61 to 67 % of the issue slots used.
#include "dt_common.cuh"
#include "dt_internal.h"
#include "train_common.cuh"

namespace dtk {

namespace {

// 16-bit rows of vectors are fetched before their turn, others where they are used:
// fp32 rows held ahead take the registers of one block in four (forward, rows of vectors,
// both norms: 15.3 us against 18.4 for 4,257 rows of 1,024, 22.8 against 26.7 for 1,200 of
// 4,096, but 71.0 against 67.3 for 36,864 of 768; element by element 16 against 21 for
// 4,257 of 1,001).
template <int DT, bool VEC>
constexpr bool kAhead = VEC && DT != 2;

// The forward pass holds one row ahead in registers (two tensors, four registers
// each; a ring as below took 90.3 us instead of 88.3, 96 x 768 rows of 768).  The
// backward pass, with four tensors, has several rows on their way into shared memory
// (131 us, 137 with one row in registers): each thread copies its own eight columns
// and reads only those back, so a copy needs no barrier, and what is in flight takes
// no registers.  kDepth: rows of a ring in a block of MAXT threads.
constexpr int kRingTensors = 4, kRingBytes = 128 << 10;
template <int MAXT>
constexpr int kDepth = kRingBytes / (kRingTensors * 16 * MAXT);
static_assert(kDepth<512> == 4 && kDepth<1024> == 2);

template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int DT>
struct RowRing {
  using T = typename TrainElem<DT>::T;
  uint4* mine;  // the thread's place in the first slot
  int c, n;     // its first column, the width
  __device__ __forceinline__ void copy(int slot, const T* __restrict__ row) const {
    if (c < n)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(mine + slot * blockDim.x)),
                   "l"(row + c)
                   : "memory");
  }
  // Columns at or past n read as 0.
  __device__ __forceinline__ void get(int slot, float (&v)[8]) const {
    const uint4 u = c < n ? mine[slot * blockDim.x] : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<DT == 0>::to_f2(q[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};

constexpr int kSums = 3;      // row sums taken together, at most
constexpr int kMaxGroups = 16;  // rows of a block

// Sums of N values over the row's warps.  Slots alternate between two halves of
// `red`, so one barrier is enough: a slot is written again two sums later, and the
// sum between has passed a barrier after every read of it.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& turn, int wpr, int w, int lane, int bar) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (wpr == 1) return;
  float* slot = red + turn * (32 * kSums);
  turn ^= 1;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slot[w * kSums + i] = v[i];
  named_bar_sync(bar, wpr * 32);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int k = 0; k < wpr; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += slot[k * kSums + i];
}

struct RowPlace {
  int w, lane, group, groups, bar;
  float* red;
};

__device__ __forceinline__ RowPlace place(int wpr, float* red_all) {
  RowPlace r;
  const int warp = threadIdx.x >> 5;
  r.group = warp / wpr;
  r.groups = (int)(blockDim.x >> 5) / wpr;
  r.w = warp - r.group * wpr;
  r.lane = threadIdx.x & 31;
  r.bar = 1 + r.group;
  r.red = red_all + r.group * (64 * kSums);  // (only rows of several warps use it: at most 8 of them a block)
  return r;
}

// A row of H columns is ceil(H / 256) warps' (one warp for rows of up to 1024, four
// pieces of eight columns a lane, took 127 us where three take 104 us: 96 x 768 rows
// of 768, both norms and a gate).  The weights come from L1 each time, in favour of
// the next row's registers.  MAXT: the block's largest size; of blocks of 256, three
// (rows held ahead) or four have to fit an SM, which caps a thread's registers (96 x
// 768 rows of 768: 88 us with three, 94 with four, 170 with five; 4,257 fp32 rows of
// 1,001: 17 us with three, 16 with four).
template <int DT, bool VEC, bool POST, bool DROP, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > 256 ? 1 : kAhead<DT, VEC> ? 3 : 4)
    residual_norm_fwd_kernel(const __grid_constant__ ResidualNormParams p) {
  using T = typename TrainElem<DT>::T;
  __shared__ float red_all[8 * 64 * kSums];
  const RowPlace at = place(p.wpr, red_all);
  int turn = 0;
  const int w = at.w, lane = at.lane, H = p.H;
  DropKey key{};
  if constexpr (DROP) key = drop_key(p.rng, p.site);
  const unsigned per_row = (unsigned)(H + 7) >> 3;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* gate = static_cast<const T*>(p.gate);
  const T* w_pre = static_cast<const T*>(p.w_pre);
  const T* w_post = static_cast<const T*>(p.w_post);
  const float inv_h = 1.f / (float)H;
  // What x^ is multiplied with on its way into h: alpha * gate * w_post / (1 - p).  Held, unless the gate's
  // row changes with the row.
  const bool fixed_gate = !gate || p.gate_rows == p.M;
  F8 cw, wpre;
  auto weigh = [&](long long gate_row) {
    cw.set(DROP ? p.alpha * p.inv_keep : p.alpha);
    F8 f;
    if constexpr (POST) {
      f.load<DT, VEC>(w_post, w, lane, H);
#pragma unroll
      for (int i = 0; i < 4; ++i) cw.p[i] = fmul2(cw.p[i], f.p[i]);
    }
    if (gate) {
      f.load<DT, VEC>(gate + gate_row * p.gate_stride, w, lane, H);
#pragma unroll
      for (int i = 0; i < 4; ++i) cw.p[i] = fmul2(cw.p[i], f.p[i]);
    }
  };
  if (fixed_gate) weigh(0);
  wpre.load<DT, VEC>(w_pre, w, lane, H);
  Raw8<DT, VEC> nx, nr;
  auto fetch = [&](long long row) {
    if (row >= p.M) return;
    nx.load(x + row * p.x_stride, w, lane, H);
    if (res) nr.load(res + row * p.res_stride, w, lane, H);
  };
  const long long step = (long long)gridDim.x * at.groups;
  long long row = (long long)blockIdx.x * at.groups + at.group;
  if constexpr (kAhead<DT, VEC>) fetch(row);
  for (; row < p.M; row += step) {
    F8 v, h;
    h.set(0.f);
    if constexpr (kAhead<DT, VEC>) {
      nx.get(v.as());
      if (res) nr.get(h.as());
      fetch(row + step);
    } else {
      v.load<DT, VEC>(x + row * p.x_stride, w, lane, H);
      if (res) h.load<DT, VEC>(res + row * p.res_stride, w, lane, H);
    }
    if (!fixed_gate) weigh(p.by_gate((int)row));
    if constexpr (POST) {
      float2 q = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) q = ffma2(v.p[i], v.p[i], q);
      float ss[1] = {both_sum(q)};
      row_sums<1>(ss, at.red, turn, p.wpr, w, lane, at.bar);
      const float r = rsqrtf(fmaf(ss[0], inv_h, p.eps));
      if (w == 0 && lane == 0) p.stats[2 * row] = r;
#pragma unroll
      for (int i = 0; i < 4; ++i) v.p[i] = fmul2(v.p[i], both(r));
    }
    if constexpr (DROP) v.keep(keep8<VEC>(key, (unsigned long long)row * per_row, w, lane, p.threshold));
    float2 q = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h.p[i] = ffma2(v.p[i], cw.p[i], h.p[i]);
      q = ffma2(h.p[i], h.p[i], q);
    }
    store8<DT, VEC>(static_cast<T*>(p.h) + row * H, w, lane, H, h.as());
    float ss[1] = {both_sum(q)};
    row_sums<1>(ss, at.red, turn, p.wpr, w, lane, at.bar);
    const float r = rsqrtf(fmaf(ss[0], inv_h, p.eps));
    if (w == 0 && lane == 0) p.stats[2 * row + 1] = r;
#pragma unroll
    for (int i = 0; i < 4; ++i) h.p[i] = fmul2(fmul2(h.p[i], both(r)), wpre.p[i]);
    store8<DT, VEC>(static_cast<T*>(p.n) + row * H, w, lane, H, h.as());
  }
}

// Adds the groups' accumulators (fixed order) and writes the block's row of
// them: fp32 into `part`, or the finished gradient into `out`.
template <int DT, bool VEC>
__device__ __forceinline__ void flush_row(float (&acc)[8], float* sh, const RowPlace& at, int H, float* part,
                                          typename TrainElem<DT>::T* out) {
  __syncthreads();  // earlier readers of `sh` are done
  const int width = at.groups > 1 ? (int)(blockDim.x / at.groups) * 8 : 0;
  if (at.groups > 1) {
    if (at.group > 0) {
      float* mine = sh + (at.group - 1) * width + at.w * 256;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i * 32 + at.lane] = acc[i];
    }
    __syncthreads();
    if (at.group == 0)
      for (int q = 1; q < at.groups; ++q) {
        const float* theirs = sh + (q - 1) * width + at.w * 256;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += theirs[i * 32 + at.lane];
      }
  }
  if (at.group == 0) {
    if (part)
      store8<2, VEC>(part, at.w, at.lane, H, acc);
    else
      store8<DT, VEC>(out, at.w, at.lane, H, acc);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
}

// Rows are cut into spans (the rows that share a row of the gate; all rows when
// there is no gate or each row has its own) and these into chunks; a block walks
// chunks blockIdx.x, blockIdx.x + gridDim.x, ... and flushes the gate's sum at
// the end of each, the weights' sums at its own end.
// MAXT: the block's largest size (a bound on the registers a thread may take).
template <int DT, bool VEC, bool POST, bool DROP, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) residual_norm_bwd_kernel(const __grid_constant__ ResidualNormParams p) {
  using T = typename TrainElem<DT>::T;
  __shared__ float red_all[8 * 64 * kSums];
  __shared__ float sums[(kMaxGroups - 1) * 256];
  const RowPlace at = place(p.wpr, red_all);
  int turn = 0;
  const int w = at.w, lane = at.lane, H = p.H;
  DropKey key{};
  if constexpr (DROP) key = drop_key(p.rng, p.site);
  const unsigned per_row = (unsigned)(H + 7) >> 3;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const T* gate = static_cast<const T*>(p.gate);
  const T* dh = static_cast<const T*>(p.dh);
  const T* dn = static_cast<const T*>(p.dn);
  T* dgate = static_cast<T*>(p.dgate);
  const T* w_post = static_cast<const T*>(p.w_post);
  // cw: alpha * gate * w_post / (1 - p), what x^ is multiplied with on its way into h.  With md the kept part of
  // D, both d(w_post) and d(gate) are multiples of sum md x^ as long as the gate's row stays: one sum (q) serves.
  F8 wpre, cw, a_pre, a_post, q;
  wpre.load<DT, VEC>(static_cast<const T*>(p.w_pre), w, lane, H);
  a_pre.set(0.f);
  a_post.set(0.f);
  q.set(0.f);
  const float inv_h = 1.f / (float)H, ak = DROP ? p.alpha * p.inv_keep : p.alpha;
  const bool sum_gate = gate && p.gate_rows > 1, row_gate = gate && p.gate_rows == 1;
  auto weigh = [&](long long gate_row) {
    cw.set(ak);
    F8 f;
    if constexpr (POST) {
      f.load<DT, VEC>(w_post, w, lane, H);
#pragma unroll
      for (int i = 0; i < 4; ++i) cw.p[i] = fmul2(cw.p[i], f.p[i]);
    }
    if (gate) {
      f.load<DT, VEC>(gate + gate_row * p.gate_stride, w, lane, H);
#pragma unroll
      for (int i = 0; i < 4; ++i) cw.p[i] = fmul2(cw.p[i], f.p[i]);
    }
  };
  if (!gate) weigh(0);

  extern __shared__ uint4 ring_smem[];
  constexpr int DEPTH = kDepth<MAXT>;
  const RowRing<DT> ring{ring_smem + threadIdx.x, (w * 32 + lane) * 8, H};
  auto fetch = [&](int stage, long long row, long long end) {
    if (row < end) {
      ring.copy(stage * 4, x + row * p.x_stride);
      if (res) ring.copy(stage * 4 + 1, res + row * p.res_stride);
      if (dh) ring.copy(stage * 4 + 2, dh + row * p.dh_stride);
      if (dn) ring.copy(stage * 4 + 3, dn + row * p.dn_stride);
    }
    copies_commit();
  };
  float n_post = 1.f, n_pre = 0.f;
  auto fetch_stats = [&](long long row) {
    if constexpr (POST) n_post = p.stats[2 * row];
    n_pre = p.stats[2 * row + 1];
  };
  for (long long chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    const long long span = chunk / p.chunks_per_span;  // the gate's row, when several rows share it
    const long long r0 = span * p.span_rows + (chunk - span * p.chunks_per_span) * p.chunk_rows;
    const long long r1 = min(r0 + p.chunk_rows, (span + 1) * p.span_rows);
    if (sum_gate) weigh(span);
    long long row = r0 + at.group;
    int stage = 0;
    if (row < r1) fetch_stats(row);
    if constexpr (kAhead<DT, VEC>)
#pragma unroll
      for (int s = 0; s < DEPTH; ++s) fetch(s, row + s * at.groups, r1);
    for (; row < r1; row += at.groups) {
      F8 xn, h, e, t;
      h.set(0.f);
      e.set(0.f);
      t.set(0.f);
      if constexpr (kAhead<DT, VEC>) {
        copies_wait<DEPTH - 1>();
        ring.get(stage * 4, xn.as());
        if (res) ring.get(stage * 4 + 1, h.as());
        if (dh) ring.get(stage * 4 + 2, e.as());
        if (dn) ring.get(stage * 4 + 3, t.as());
        fetch(stage, row + DEPTH * at.groups, r1);
        stage = stage + 1 == DEPTH ? 0 : stage + 1;
      } else {
        xn.load<DT, VEC>(x + row * p.x_stride, w, lane, H);
        if (res) h.load<DT, VEC>(res + row * p.res_stride, w, lane, H);
        if (dh) e.load<DT, VEC>(dh + row * p.dh_stride, w, lane, H);
        if (dn) t.load<DT, VEC>(dn + row * p.dn_stride, w, lane, H);
      }
      const float r_post = n_post, r_pre = n_pre;
      if (row + at.groups < r1) fetch_stats(row + at.groups);
      if (row_gate) weigh(row);
      uint32_t m = 0xffu;
      if constexpr (DROP) m = keep8<VEC>(key, (unsigned long long)row * per_row, w, lane, p.threshold);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0, s2 = s0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (POST) xn.p[i] = fmul2(xn.p[i], both(r_post));  // from here on the normalised x
        // Dropped: x itself without a post norm (it counts as 0 whatever it was, in the gate's gradient as well).
        auto drop = [&](float2& v) {
          v.x = (m >> (2 * i)) & 1u ? v.x : 0.f;
          v.y = (m >> (2 * i + 1)) & 1u ? v.y : 0.f;
        };
        if constexpr (DROP && !POST) drop(xn.p[i]);
        float2 gv = fmul2(xn.p[i], cw.p[i]);
        if constexpr (DROP && POST) drop(gv);
        h.p[i] = fmul2(fadd2(h.p[i], gv), both(r_pre));  // the normalised h
        a_pre.p[i] = ffma2(t.p[i], h.p[i], a_pre.p[i]);
        t.p[i] = fmul2(t.p[i], wpre.p[i]);
        e.p[i] = ffma2(t.p[i], both(r_pre), e.p[i]);
        s0 = ffma2(t.p[i], h.p[i], s0);
        if constexpr (POST) {
          s1 = ffma2(gv, e.p[i], s1);
          s2 = ffma2(gv, h.p[i], s2);
        }
      }
      float s[3] = {both_sum(s0), both_sum(s1), both_sum(s2)};
      if constexpr (POST) {
        row_sums<3>(s, at.red, turn, p.wpr, w, lane, at.bar);
      } else {
        float one[1] = {s[0]};
        row_sums<1>(one, at.red, turn, p.wpr, w, lane, at.bar);
        s[0] = one[0];
      }
      const float rc = r_pre * s[0] * inv_h, c_post = (s[1] - rc * s[2]) * inv_h * r_post;
#pragma unroll
      for (int i = 0; i < 4; ++i) e.p[i] = ffma2(h.p[i], both(-rc), e.p[i]);  // the gradient of h
      if (p.dresidual) store8<DT, VEC>(static_cast<T*>(p.dresidual) + row * H, w, lane, H, e.as());
      if constexpr (DROP) e.keep(m);
      if (row_gate) {
        // The gate's row is this row's own.
        F8 f;
        f.set(ak);
        if constexpr (POST) {
          F8 g;
          f.load<DT, VEC>(w_post, w, lane, H);
          g.load<DT, VEC>(gate + row * p.gate_stride, w, lane, H);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f.p[i] = fmul2(f.p[i], both(ak));
            a_post.p[i] = ffma2(fmul2(g.p[i], both(ak)), fmul2(e.p[i], xn.p[i]), a_post.p[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) f.p[i] = fmul2(f.p[i], fmul2(xn.p[i], e.p[i]));
        store8<DT, VEC>(dgate + row * H, w, lane, H, f.as());
      } else if (POST || sum_gate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q.p[i] = ffma2(e.p[i], xn.p[i], q.p[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e.p[i] = fmul2(e.p[i], cw.p[i]);
        if constexpr (POST) e.p[i] = ffma2(e.p[i], both(r_post), fmul2(xn.p[i], both(-c_post)));
      }
      store8<DT, VEC>(static_cast<T*>(p.dx) + row * H, w, lane, H, e.as());
    }
    if (sum_gate) {
      // The span's sum, as the gate's gradient and as a share of the weight's.
      F8 f;
      if constexpr (POST) {
        f.load<DT, VEC>(gate + span * p.gate_stride, w, lane, H);
#pragma unroll
        for (int i = 0; i < 4; ++i) a_post.p[i] = ffma2(fmul2(f.p[i], both(ak)), q.p[i], a_post.p[i]);
        f.load<DT, VEC>(w_post, w, lane, H);
#pragma unroll
        for (int i = 0; i < 4; ++i) q.p[i] = fmul2(q.p[i], fmul2(f.p[i], both(ak)));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) q.p[i] = fmul2(q.p[i], both(ak));
      }
      const bool whole = p.chunks_per_span == 1;
      flush_row<DT, VEC>(q.as(), sums, at, H, whole ? nullptr : p.part_gate + chunk * H, whole ? dgate + span * H : nullptr);
    }
  }
  if constexpr (POST) {
    if (!gate)
#pragma unroll
      for (int i = 0; i < 4; ++i) a_post.p[i] = fmul2(q.p[i], both(ak));
  }
  const bool alone = gridDim.x == 1;
  if (dn)
    flush_row<DT, VEC>(a_pre.as(), sums, at, H, alone ? nullptr : p.part_pre + (long long)blockIdx.x * H,
                       static_cast<T*>(p.dw_pre));
  if constexpr (POST)
    flush_row<DT, VEC>(a_post.as(), sums, at, H, alone ? nullptr : p.part_post + (long long)blockIdx.x * H,
                       static_cast<T*>(p.dw_post));
}

// Adds partial rows in a fixed order: out[j][c] = sum over i < n of
// part[(j * n + i) * H + c].  The weights' gradients have one row of many parts:
// 32 columns a block, 32 slices of the parts, then a shuffle tree.  So has a
// gate's when few rows share many parts; else (narrow) a warp takes 32 columns of a row.
struct SumJob {
  const float* part;
  void* out;
  long long n, rows;  // partial rows of each output row; output rows
};
template <int DT>
__global__ void __launch_bounds__(1024) sum_rows_kernel(SumJob w0, SumJob w1, SumJob gate, int H) {
  using T = typename TrainElem<DT>::T;
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  if (blockIdx.y >= 2 && gate.n < 32) {
    const long long j = (long long)(blockIdx.y - 2) * 32 + slice;
    if (j >= gate.rows || col >= H) return;
    const float* q = gate.part + j * gate.n * H + col;
    float s = 0.f;
#pragma unroll 4
    for (long long i = 0; i < gate.n; ++i) s += q[i * H];
    static_cast<T*>(gate.out)[j * H + col] = TrainElem<DT>::from_f(s);
    return;
  }
  SumJob job = blockIdx.y == 0 ? w0 : blockIdx.y == 1 ? w1 : gate;
  if (!job.part) return;
  const long long j = blockIdx.y < 2 ? 0 : blockIdx.y - 2;
  job.part += j * job.n * H;
  float s = 0.f;
  if (col < H) {
    const float* q = job.part + col;
#pragma unroll 4
    for (long long i = slice; i < job.n; i += 32) s += q[i * H];
  }
  sh[slice][lane] = s;
  __syncthreads();
  // Warp k adds column k's slices.
  s = sh[lane][slice];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && blockIdx.x * 32 + slice < H)
    static_cast<T*>(job.out)[j * H + blockIdx.x * 32 + slice] = TrainElem<DT>::from_f(s);
}

template <int DT, bool VEC, bool POST, int MAXT>
cudaError_t run_fwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  if (p.threshold)
    residual_norm_fwd_kernel<DT, VEC, POST, true, MAXT><<<grid, block, 0, st>>>(p);
  else
    residual_norm_fwd_kernel<DT, VEC, POST, false, MAXT><<<grid, block, 0, st>>>(p);
  return cudaGetLastError();
}
template <int DT, bool VEC, bool POST>
cudaError_t launch_fwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  return block > 256 ? run_fwd<DT, VEC, POST, 1024>(p, grid, block, st) : run_fwd<DT, VEC, POST, 256>(p, grid, block, st);
}

template <int DT, bool VEC, bool POST, int MAXT>
cudaError_t run_bwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  auto kern = p.threshold ? residual_norm_bwd_kernel<DT, VEC, POST, true, MAXT>
                          : residual_norm_bwd_kernel<DT, VEC, POST, false, MAXT>;
  unsigned smem = 0;
  if constexpr (kAhead<DT, VEC>) {
    smem = kDepth<MAXT> * kRingTensors * 16 * block;
    const cudaError_t e = smem_limit_once(reinterpret_cast<const void*>(kern), kRingBytes);
    if (e != cudaSuccess) return e;
  }
  kern<<<grid, block, smem, st>>>(p);
  return cudaGetLastError();
}
template <int DT, bool VEC, bool POST>
cudaError_t launch_bwd(const ResidualNormParams& p, unsigned grid, unsigned block, cudaStream_t st) {
  return block > 512 ? run_bwd<DT, VEC, POST, 1024>(p, grid, block, st) : run_bwd<DT, VEC, POST, 512>(p, grid, block, st);
}

// 16-byte accesses need every row on a 16-byte boundary and whole vectors.
bool can_vector(const ResidualNormParams& p, int dtype, bool bwd) {
  const long long e = dtype == 2 ? 4 : 2;
  if (p.H % 8) return false;
  const void* ptrs[] = {p.x, p.residual, p.gate, p.w_pre, p.w_post, bwd ? p.dh : p.h, bwd ? p.dn : p.n, p.dx,
                        p.dresidual, p.dgate, p.dw_pre, p.dw_post};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return false;
  const long long strides[] = {p.x_stride, p.residual ? p.res_stride : 0, p.gate ? p.gate_stride : 0,
                               p.dh ? p.dh_stride : 0, p.dn ? p.dn_stride : 0};
  for (long long s : strides)
    if (s * e % 16) return false;
  return true;
}

}  // namespace

// Warps that hold a row (eight columns a thread), and rows that a block of up to
// `warps` warps holds.
static int rn_wpr(int H) { return (H + 255) / 256; }
static int rn_groups(int H, int warps) { return rn_wpr(H) >= warps ? 1 : warps / rn_wpr(H); }
// Warps of a block of the backward pass: with a ring of rows on their way one block of
// 16 warps fills an SM, without one two blocks of 8 (up to 128 registers a thread; planned
// for four, the grid ran in two waves and left twice the parts: 48 x 768 fp32 rows of 768
// 139 + 7 us instead of 125 + 4, 4,257 of 1,001 27.5 + 4.4 instead of 26 + 3.3).
constexpr int kFwdWarps = 8;
static int rn_bwd_warps(bool ring) { return ring ? 16 : 8; }

// Chunks of the backward pass: one for each block that the GPU holds, never across
// two spans.  gate_rows: rows that share a row of the gate, 0 without one.
ResidualNormPlan residual_norm_plan(long long M, int H, long long gate_rows, bool ring, int num_sms) {
  ResidualNormPlan q;
  const int groups = rn_groups(H, rn_bwd_warps(ring)), warps = groups * rn_wpr(H);
  q.groups = groups;
  q.span_rows = gate_rows > 1 ? gate_rows : M;
  const long long spans = M / q.span_rows;
  const int fit = 16 / warps;  // blocks on an SM
  const long long want = (long long)num_sms * (fit < 1 ? 1 : fit);
  const long long most = (q.span_rows + groups - 1) / groups;
  long long per_span = want / spans;
  if (per_span > most) per_span = most;
  if (per_span < 1) per_span = 1;
  q.chunk_rows = (q.span_rows + per_span - 1) / per_span;
  q.chunks_per_span = (q.span_rows + q.chunk_rows - 1) / q.chunk_rows;
  q.chunks = spans * q.chunks_per_span;
  q.grid = q.chunks < want ? q.chunks : want;
  return q;
}

cudaError_t launch_residual_norm_fwd_sm100(ResidualNormParams p, int dtype, int num_sms, cudaStream_t st) {
  p.wpr = rn_wpr(p.H);
  const int groups = rn_groups(p.H, kFwdWarps);
  const unsigned block = (unsigned)(p.wpr * groups * 32);
  const long long want = (p.M + groups - 1) / groups, cap = (long long)num_sms * 32;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  const bool vec = can_vector(p, dtype, false), post = p.w_post != nullptr;
#define DT_FWD(DT)                                                                             \
  return vec ? (post ? launch_fwd<DT, true, true>(p, grid, block, st) : launch_fwd<DT, true, false>(p, grid, block, st)) \
             : (post ? launch_fwd<DT, false, true>(p, grid, block, st) : launch_fwd<DT, false, false>(p, grid, block, st))
  if (dtype == 0) DT_FWD(0);
  if (dtype == 1) DT_FWD(1);
  DT_FWD(2);
#undef DT_FWD
}

bool residual_norm_ring(const ResidualNormParams& p, int dtype) { return dtype != 2 && can_vector(p, dtype, true); }

cudaError_t launch_residual_norm_bwd_sm100(ResidualNormParams p, const ResidualNormPlan& plan, int dtype,
                                           cudaStream_t st) {
  p.wpr = rn_wpr(p.H);
  const unsigned block = (unsigned)(p.wpr * plan.groups * 32), grid = (unsigned)plan.grid;
  p.chunks = plan.chunks;
  p.chunk_rows = plan.chunk_rows;
  p.chunks_per_span = plan.chunks_per_span;
  p.span_rows = plan.span_rows;
  const bool sum_gate = p.gate && p.gate_rows > 1;
  const bool vec = can_vector(p, dtype, true), post = p.w_post != nullptr;
  cudaError_t e;
#define DT_BWD(DT)                                                                             \
  e = vec ? (post ? launch_bwd<DT, true, true>(p, grid, block, st) : launch_bwd<DT, true, false>(p, grid, block, st)) \
          : (post ? launch_bwd<DT, false, true>(p, grid, block, st) : launch_bwd<DT, false, false>(p, grid, block, st))
  if (dtype == 0) DT_BWD(0);
  else if (dtype == 1) DT_BWD(1);
  else DT_BWD(2);
#undef DT_BWD
  if (e != cudaSuccess) return e;
  // What the blocks left in parts.
  SumJob w0{}, w1{}, gate{};
  if (grid > 1 && p.dn) w0 = SumJob{p.part_pre, p.dw_pre, (long long)grid, 1};
  if (grid > 1 && post) w1 = SumJob{p.part_post, p.dw_post, (long long)grid, 1};
  if (sum_gate && plan.chunks_per_span > 1)
    gate = SumJob{p.part_gate, p.dgate, plan.chunks_per_span, plan.chunks / plan.chunks_per_span};
  if (!w0.part && !w1.part && !gate.part) return cudaSuccess;
  const dim3 g((unsigned)((p.H + 31) / 32), (unsigned)(2 + (gate.n < 32 ? (gate.rows + 31) / 32 : gate.rows)));
  if (dtype == 0) sum_rows_kernel<0><<<g, 1024, 0, st>>>(w0, w1, gate, p.H);
  else if (dtype == 1) sum_rows_kernel<1><<<g, 1024, 0, st>>>(w0, w1, gate, p.H);
  else sum_rows_kernel<2><<<g, 1024, 0, st>>>(w0, w1, gate, p.H);
  return cudaGetLastError();
}

}  // namespace dtk
