// The norms around a block of a residual network, fused with its gate and residual scale, forward and backward (f32 or
// bf16 rows; statistics, weights and every sum in f32). With rms(z) = z / sqrt(mean z^2 + eps), a = sigmoid(gate):
//
//   forward   bh = rms(branch) (or branch), r = x + s a w1 bh, y = w2 rms(r)
//   backward  rh = r rstd, g = dy w2, d = dr + rstd (g - rh mean(g rh)); dx = d
//             dgate = s d w1 bh a (1 - a), t = s d a w1, dbranch = rstd_b (t - bh mean(t bh))
//             dw1 = sum_rows s d a bh, dw2 = sum_rows dy rh
//
// The second norm is of r as it is stored (rounded to the rows' type), which is also what the way back has in hand.
//
// Bound by HBM: 4 or 5 (forward), 6 to 8 (backward) passes over rows x cols values. As in the layer norm, a row is read
// once and stays in the registers of TPR threads, thread t holding its columns (k TPR + t) VEC + j, with 16-byte loads
// where bases, row strides and the width allow them; persistent blocks keep the weights in registers and load the next
// row while they fold the current one. Each direction folds twice per row, one after the other: the second norm needs
// the first one's result.
//
// Measured, 65,536 x 2,048 bf16 with gate: 211 to 234 us forward (97 to 88 % of a copy's 6,545 GB/s), 424 back (77 %); without a
// gate 177 and 284; f32 with gate 396 and 646 (the copy's rate). Back, rows of 4,096, 8,192 and 16,384 bf16 columns, a cluster
// of blocks each, reach 73, 68 and 59 %.
#include <atomic>
#include "pl_rows.cuh"
#include "pl_runtime.h"
#include "pl_tc.cuh"

namespace pl {

// sigmoid(g), and with it 1 - sigmoid(g), for rows of type T. The fast exponential is 2^-21 + |g| 2^-23 of its value off, which the
// rounding of bf16 rows, 2^-8, hides; f32 rows get the exact one, and 6 units of 2^-23 at any g. The division is 2 units off at
// most, and zero where sigmoid(g) is below 2^-126.
template <typename T>
__device__ __forceinline__ void sigmoid2(float g, float& a, float& na) {
  const float t = sizeof(T) == 2 ? __expf(-g) : expf(-g);  // infinite where sigmoid(g) is zero
  a = __fdividef(1.f, 1.f + t);
  na = g >= 0.f ? t * a : 1.f - a;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  float a, na;
  sigmoid2<T>(g, a, na);
  return a;
}

template <typename T>
struct BlockArgs {  // forward
  const T *x, *branch, *gate;
  long ldx, ldb, ldg;
  const float *w1, *w2;
  float scale, eps;
  long rows, cols;
  T *r, *y;
  long ldr, ldy;
  float *rstd_b, *rstd;  // rstd_b: NULL without the first norm
};

template <typename T, int VEC, int TPR, int K, bool GATE>
__global__ void __launch_bounds__(norm_threads(TPR), norm_blocks(TPR)) block_fwd_kernel(const BlockArgs<T> p) {
  grid_wait();
  grid_next();
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  __shared__ float scr[2][2][32];  // [row parity][fold]
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv = 1.f / (float)p.cols;
  const long step = (long)gridDim.x * G;
  Vec<VEC> w1[K], w2[K];
  bool in_row[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const long c = (long)(k * TPR + t) * VEC;
    in_row[k] = c < p.cols;
    w1[k] = w2[k] = vall<VEC>(1.f);
    if (p.w1 && in_row[k]) load_param<VEC>(p.w1, c, w1[k].v);
    if (p.w2 && in_row[k]) load_param<VEC>(p.w2, c, w2[k].v);
    w1[k] = vmul(w1[k], vall<VEC>(p.scale));
  }
  Pack<T, VEC> nx[K], nb[K], ng[GATE ? K : 1];
  auto load = [&](long row) {  // what lies outside the matrix reads as zero
#pragma unroll
    for (int k = 0; k < K; k++) {
      const long c = (long)(k * TPR + t) * VEC;
      if (row < p.rows && in_row[k]) {
        nb[k].load(p.branch + row * p.ldb + c);
        nx[k].load(p.x + row * p.ldx + c);
        if constexpr (GATE) ng[k].load(p.gate + row * p.ldg + c);
      } else {
        nx[k] = nb[k] = narrow<T, VEC>(vall<VEC>(0.f));
        if constexpr (GATE) ng[k] = nx[k];
      }
    }
  };
  load((long)blockIdx.x * G + g);
  int parity = 0;
  for (long base = (long)blockIdx.x * G; base < p.rows; base += step, parity ^= 1) {
    const long row = base + g;
    Vec<VEC> x[K], b[K];
    Vec<VEC> s = vall<VEC>(0.f);
#pragma unroll
    for (int k = 0; k < K; k++) {
      x[k] = widen<T, VEC>(nx[k]);
      b[k] = widen<T, VEC>(nb[k]);
      s = vfma(b[k], b[k], s);
      b[k] = vmul(b[k], w1[k]);
      if constexpr (GATE) {
        const Vec<VEC> f = widen<T, VEC>(ng[k]);
#pragma unroll
        for (int j = 0; j < VEC; j++) b[k].v[j] *= sigmoid<T>(f.v[j]);
      }
    }
    load(row + step);
    float rb = 1.f;
    if (p.rstd_b) {
      rb = 1.f / sqrtf(group_sum<TPR>(vsum(s), scr[parity][0]) * inv + p.eps);
      if (t == 0 && row < p.rows) p.rstd_b[row] = rb;
    }
    s = vall<VEC>(0.f);
    Pack<T, VEC> r[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
      r[k] = narrow<T, VEC>(vfma(b[k], vall<VEC>(rb), x[k]));
      x[k] = widen<T, VEC>(r[k]);
      if (in_row[k]) s = vfma(x[k], x[k], s);
    }
    const float rr = 1.f / sqrtf(group_sum<TPR>(vsum(s), scr[parity][1]) * inv + p.eps);
    if (row < p.rows) {
      if (t == 0) p.rstd[row] = rr;
#pragma unroll
      for (int k = 0; k < K; k++)
        if (in_row[k]) {
          const long c = (long)(k * TPR + t) * VEC;
          r[k].store(p.r + row * p.ldr + c);
          narrow<T, VEC>(vmul(vmul(x[k], vall<VEC>(rr)), w2[k])).store(p.y + row * p.ldy + c);
        }
    }
  }
}

// Rows too wide for the registers: one block per row, read again from L2 for each fold.
template <typename T>
__global__ void __launch_bounds__(512) block_fwd_wide_kernel(const BlockArgs<T> p) {
  grid_wait();
  grid_next();
  __shared__ float scr[2][32];
  const long row = blockIdx.x;
  const T *x = p.x + row * p.ldx, *b = p.branch + row * p.ldb, *g = p.gate ? p.gate + row * p.ldg : nullptr;
  T *r = p.r + row * p.ldr, *y = p.y + row * p.ldy;
  const float inv = 1.f / (float)p.cols;
  float rb = 1.f, s = 0.f;
  if (p.rstd_b) {
    for (long c = threadIdx.x; c < p.cols; c += 512) {
      const float f = to_f(b[c]);
      s = __fmaf_rn(f, f, s);
    }
    rb = 1.f / sqrtf(group_sum<512>(s, scr[0]) * inv + p.eps);
    if (threadIdx.x == 0) p.rstd_b[row] = rb;
  }
  s = 0.f;
  for (long c = threadIdx.x; c < p.cols; c += 512) {
    float f = to_f(b[c]) * (p.w1 ? p.w1[c] * p.scale : p.scale);
    const float a = g ? sigmoid<T>(to_f(g[c])) : 1.f;
    const T v = from_f<T>(__fmaf_rn(f * a, rb, to_f(x[c])));
    r[c] = v;
    f = to_f(v);
    s = __fmaf_rn(f, f, s);
  }
  const float rr = 1.f / sqrtf(group_sum<512>(s, scr[1]) * inv + p.eps);
  if (threadIdx.x == 0) p.rstd[row] = rr;
  for (long c = threadIdx.x; c < p.cols; c += 512) {  // a thread reads what it wrote itself
    const float f = to_f(r[c]) * rr;
    y[c] = from_f<T>(p.w2 ? f * p.w2[c] : f);
  }
}

// ---------------------------------------------------------------------------------------------- backward
template <typename T>
struct BlockGradArgs {
  const T *dr, *dy, *branch, *gate, *r;  // dr, gate may be NULL
  long lddr, lddy, ldb, ldg, ldr;
  const float *rstd_b, *rstd, *w1, *w2;
  float scale;
  long rows, cols;
  T *dx, *db, *dg;
  long lddx, lddb, lddg;
  float *part;  // [clusters][2][cols] column sums of the clusters' rows (dw1, dw2), or NULL
  long width;   // columns of a block: all, or of a cluster's block (rank width .. (rank + 1) width)
  unsigned* err;
};

// Sum over a row that C blocks of TPR threads share (a fixed order, the same in all of them). `scr` holds 32 floats, or one
// per warp of the cluster, of the block's own for this call. The warps' sums go to the other blocks' shared memory with
// their barrier's count of bytes, in its phase `phase`: a barrier of the cluster would wait for the rows' stores as well
// (32,768 x 4,096 bf16 with gate back: 591 us instead of 449).
template <int TPR, int C>
__device__ __forceinline__ float row_sum(float v, float* scr, uint64_t* bar, uint32_t phase, int rank, unsigned* err) {
  if constexpr (C == 1) {
    return group_sum<TPR>(v, scr);
  } else {
    constexpr int NW = TPR / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) tc::mbar_expect_tx(bar, C * NW * 4);
    v = warp_sum(v);
    if (lane < C)
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                       tc::cluster_addr(tc::smem_u32(scr + rank * NW + warp), lane)),
                   "r"(__float_as_uint(v)), "r"(tc::cluster_addr(tc::smem_u32(bar), lane))
                   : "memory");
    v = tc::mbar_wait(bar, phase, err, PL_ERR_MBAR_TIMEOUT) ? 0.f : __int_as_float(0x7fffffff);  // NaN: no gradient
#pragma unroll
    for (int q = 0; q < (C * NW + 31) / 32; q++)
      if (q * 32 + lane < C * NW) v += scr[q * 32 + lane];
    return warp_sum(v);
  }
}

// C: blocks per row, a cluster. A row's slot of `scr` is written again two rows later, by which time the writer has every
// warp's sum of the next row, sent behind its reads of this one.
template <typename T, int VEC, int TPR, int K, int C, bool GATE>
__global__ void __launch_bounds__(norm_threads(TPR), norm_blocks(TPR)) block_bwd_kernel(const BlockGradArgs<T> p) {
  grid_wait();
  grid_next();
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  static_assert(C == 1 || G == 1, "the rows of a cluster");
  __shared__ float scr[2][2][C * TPR / 32 > 32 ? C * TPR / 32 : 32];  // [row parity][fold]
  extern __shared__ float fold[];                                     // [G][2][TPR * VEC * K] (G > 1)
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR, rank = C > 1 ? blockIdx.x % C : 0;
  const float inv = 1.f / (float)p.cols;
  const long first = (long)(blockIdx.x / C) * G, step = (long)(gridDim.x / C) * G, c0 = rank * p.width;
  const bool has_dr = p.dr != nullptr;
  __shared__ uint64_t bar[2][2];
  if constexpr (C > 1) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < 4; i++) tc::mbar_init(&bar[i >> 1][i & 1], 1);
      tc::fence_mbar_init();
    }
    tc::cluster_sync();  // the others' barriers are there
  }
  Vec<VEC> w1[K], w2[K], s1[K], s2[K];
  bool in_row[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const long c = c0 + (k * TPR + t) * VEC;
    in_row[k] = c < p.cols && (C == 1 || c < c0 + p.width);
    s1[k] = s2[k] = vall<VEC>(0.f);
    w1[k] = w2[k] = vall<VEC>(1.f);
    if (p.w1 && in_row[k]) load_param<VEC>(p.w1, c, w1[k].v);
    if (p.w2 && in_row[k]) load_param<VEC>(p.w2, c, w2[k].v);
  }
  Pack<T, VEC> nd[K], ny[K], nb[K], nr[K], ng[GATE ? K : 1];
  float nrb, nrr;
  auto load = [&](long row) {  // what lies outside the matrix reads as zero and adds nothing to any sum
    const bool ok = row < p.rows;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const long c = c0 + (k * TPR + t) * VEC;
      nd[k] = ny[k] = nb[k] = nr[k] = narrow<T, VEC>(vall<VEC>(0.f));
      if constexpr (GATE) ng[k] = nd[k];
      if (ok && in_row[k]) {
        ny[k].load(p.dy + row * p.lddy + c);
        nr[k].load(p.r + row * p.ldr + c);
        if (has_dr) nd[k].load(p.dr + row * p.lddr + c);
        nb[k].load(p.branch + row * p.ldb + c);
        if constexpr (GATE) ng[k].load(p.gate + row * p.ldg + c);
      }
    }
    nrr = ok ? __ldg(p.rstd + row) : 0.f;
    nrb = ok ? (p.rstd_b ? __ldg(p.rstd_b + row) : 1.f) : 0.f;
  };
  load(first + g);
  int parity = 0;
  uint32_t phase = 0;  // of the barriers of this parity, a phase per use
  for (long base = first; base < p.rows; base += step, phase ^= parity, parity ^= 1) {
    const long row = base + g;
    const float rr = nrr, rb = nrb;
    Vec<VEC> d[K], rh[K], gy[K], bh[K], c1[GATE ? K : 1], c2[GATE ? K : 1];
    Vec<VEC> s = vall<VEC>(0.f);
#pragma unroll
    for (int k = 0; k < K; k++) {
      rh[k] = vmul(widen<T, VEC>(nr[k]), vall<VEC>(rr));
      gy[k] = widen<T, VEC>(ny[k]);
      s2[k] = vfma(gy[k], rh[k], s2[k]);
      gy[k] = vmul(gy[k], w2[k]);
      s = vfma(gy[k], rh[k], s);
      d[k] = widen<T, VEC>(nd[k]);
      bh[k] = vmul(widen<T, VEC>(nb[k]), vall<VEC>(rb));
      if constexpr (GATE) {  // what d is multiplied with in its way to the branch and the gate: before the fold, not behind it
        const Vec<VEC> f = widen<T, VEC>(ng[k]);
        Vec<VEC> na;
#pragma unroll
        for (int j = 0; j < VEC; j++) sigmoid2<T>(f.v[j], c1[k].v[j], na.v[j]);
        c1[k] = vmul(c1[k], vall<VEC>(p.scale));
        c2[k] = vmul(vmul(vmul(c1[k], na), bh[k]), w1[k]);
      }
    }
    if constexpr (!GATE) load(row + step);
    const float m1 = -inv * row_sum<TPR, C>(vsum(s), scr[parity][0], &bar[parity][0], phase, rank, p.err);
    s = vall<VEC>(0.f);
#pragma unroll
    for (int k = 0; k < K; k++) {
      const long c = c0 + (k * TPR + t) * VEC;
      d[k] = vfma(vfma(rh[k], vall<VEC>(m1), gy[k]), vall<VEC>(rr), d[k]);
      if (row < p.rows && in_row[k]) narrow<T, VEC>(d[k]).store(p.dx + row * p.lddx + c);
      if constexpr (GATE) {
        if (row < p.rows && in_row[k]) narrow<T, VEC>(vmul(d[k], c2[k])).store(p.dg + row * p.lddg + c);
        d[k] = vmul(d[k], c1[k]);
      } else {
        d[k] = vmul(d[k], vall<VEC>(p.scale));
      }
      s1[k] = vfma(d[k], bh[k], s1[k]);
      d[k] = vmul(d[k], w1[k]);
      s = vfma(d[k], bh[k], s);
    }
    if constexpr (GATE) load(row + step);  // (before the first fold the registers do not do for both: 470 us instead of 420)
    float m2 = 0.f;
    if (p.rstd_b) m2 = -inv * row_sum<TPR, C>(vsum(s), scr[parity][1], &bar[parity][1], phase, rank, p.err);
    if (row < p.rows)
#pragma unroll
      for (int k = 0; k < K; k++)
        if (in_row[k])
          narrow<T, VEC>(vmul(vfma(bh[k], vall<VEC>(m2), d[k]), vall<VEC>(rb)))
              .store(p.db + row * p.lddb + c0 + (k * TPR + t) * VEC);
  }
  if constexpr (C > 1) tc::cluster_sync();  // none leaves while another may still send to it
  if (!p.part) return;
  float* pw = p.part + (long)(blockIdx.x / C) * 2 * p.cols;
  if constexpr (G > 1) {
    constexpr int W = TPR * VEC * K;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const int c = (k * TPR + t) * VEC + j;
        fold[(g * 2) * W + c] = s1[k].v[j];
        fold[(g * 2 + 1) * W + c] = s2[k].v[j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < p.cols; c += THREADS) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < G; q++) {
        a += fold[(q * 2) * W + c];
        b += fold[(q * 2 + 1) * W + c];
      }
      pw[c] = a;
      pw[p.cols + c] = b;
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const long c = c0 + (k * TPR + t) * VEC + j;
        if (in_row[k]) {
          pw[c] = s1[k].v[j];
          pw[p.cols + c] = s2[k].v[j];
        }
      }
  }
}

// Rows too wide for the registers. One block per row for what goes row by row; the mean of g rh is kept for the columns'
// sums.
template <typename T>
__global__ void __launch_bounds__(512) block_bwd_wide_kernel(const BlockGradArgs<T> p, float* __restrict__ mean) {
  grid_wait();
  grid_next();
  __shared__ float scr[2][32];
  const long row = blockIdx.x;
  const T *dy = p.dy + row * p.lddy, *r = p.r + row * p.ldr, *b = p.branch + row * p.ldb;
  const T *dr = p.dr ? p.dr + row * p.lddr : nullptr, *g = p.gate ? p.gate + row * p.ldg : nullptr;
  const float inv = 1.f / (float)p.cols, rr = p.rstd[row], rb = p.rstd_b ? p.rstd_b[row] : 1.f;
  float s = 0.f;
  for (long c = threadIdx.x; c < p.cols; c += 512)
    s = __fmaf_rn(to_f(dy[c]) * (p.w2 ? p.w2[c] : 1.f), to_f(r[c]) * rr, s);
  const float m1 = group_sum<512>(s, scr[0]) * inv;
  if (mean && threadIdx.x == 0) mean[row] = m1;
  auto at = [&](long c, float& bh, float& a, float& na) {
    bh = to_f(b[c]) * rb;
    a = 1.f;
    na = 0.f;
    if (g) sigmoid2<T>(to_f(g[c]), a, na);
    const float gy = to_f(dy[c]) * (p.w2 ? p.w2[c] : 1.f);
    return (dr ? to_f(dr[c]) : 0.f) + (gy - to_f(r[c]) * rr * m1) * rr;
  };
  s = 0.f;
  for (long c = threadIdx.x; c < p.cols; c += 512) {
    float bh, a, na;
    const float d = at(c, bh, a, na), w = p.w1 ? p.w1[c] : 1.f, t = d * p.scale * a * w;
    p.dx[row * p.lddx + c] = from_f<T>(d);
    if (g) p.dg[row * p.lddg + c] = from_f<T>(t * na * bh);
    s = __fmaf_rn(t, bh, s);
  }
  const float m2 = p.rstd_b ? group_sum<512>(s, scr[1]) * inv : 0.f;
  for (long c = threadIdx.x; c < p.cols; c += 512) {
    float bh, a, na;
    const float d = at(c, bh, a, na), w = p.w1 ? p.w1[c] : 1.f;
    p.db[row * p.lddb + c] = from_f<T>((d * p.scale * a * w - bh * m2) * rb);
  }
}
// dw1, dw2: one thread per column and slice of the rows, [gridDim.y][2][cols] parts.
template <typename T>
__global__ void __launch_bounds__(256)
    block_bwd_wide_param_kernel(const BlockGradArgs<T> p, const float* __restrict__ mean) {
  grid_wait();
  grid_next();
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.cols) return;
  const float w2 = p.w2 ? p.w2[c] : 1.f;
  float s1 = 0.f, s2 = 0.f;
  for (long row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float rr = p.rstd[row], rh = to_f(p.r[row * p.ldr + c]) * rr, dy = to_f(p.dy[row * p.lddy + c]);
    const float a = p.gate ? sigmoid<T>(to_f(p.gate[row * p.ldg + c])) : 1.f;
    const float d = (p.dr ? to_f(p.dr[row * p.lddr + c]) : 0.f) + (dy * w2 - rh * mean[row]) * rr;
    s1 = __fmaf_rn(d * p.scale * a, to_f(p.branch[row * p.ldb + c]) * (p.rstd_b ? p.rstd_b[row] : 1.f), s1);
    s2 = __fmaf_rn(dy, rh, s2);
  }
  float* q = p.part + (long)blockIdx.y * 2 * p.cols;
  q[c] = s1;
  q[p.cols + c] = s2;
}

// ---------------------------------------------------------------------------------------------- host side
constexpr long kBlockMost = 16384;  // the widest row that stays in registers
constexpr int kWideSlices = 64;     // of the rows, for the column sums of wider ones

template <typename T, int VEC, int TPR, int K, bool GATED = true>
static int fwd_launch(const BlockArgs<T>& p, cudaStream_t st) {
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  const long need = ceil_div(p.rows, G), most = (long)kNormSms * norm_blocks(TPR);
  const unsigned grid = (unsigned)(need < most ? need : most);
  auto kernel = block_fwd_kernel<T, VEC, TPR, K, false>;
  if constexpr (GATED)
    if (p.gate) kernel = block_fwd_kernel<T, VEC, TPR, K, true>;
  PL_CUDA(launch_early(kernel, grid, THREADS, 0, st, p));
  count_launch();
  return PL_OK;
}
// Clusters of the kernel that the device holds at once, or 0 where it does not say. More in the grid than these would run when
// the first are done, a whole share of the rows later: 37 clusters of four blocks, an SM each, leave four to a second turn
// (8,192 x 16,384 bf16 with gate: 897 us, with the 33 that fit 558).
static int resident_clusters(const void* kernel, std::atomic<int>* known, cudaLaunchConfig_t cfg, int c) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if ((n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  cfg.gridDim = (unsigned)c;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 0;
  }
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}
template <typename T, int VEC, int TPR, int K, int C, bool GATE>
static int bwd_launch(BlockGradArgs<T>& p, float* dw1, float* dw2, cudaStream_t st) {
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  constexpr size_t FOLD = G > 1 ? (size_t)G * 2 * TPR * VEC * K * 4 : 0;
  static_assert(FOLD <= 48 * 1024, "column sums of the groups");
  auto kernel = block_bwd_kernel<T, VEC, TPR, K, C, GATE>;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = THREADS;
  cfg.dynamicSmemBytes = FOLD;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  const long need = ceil_div(p.rows, G);
  long most = (long)kNormSms * norm_blocks(TPR) / C;
  if constexpr (C > 1) {
    static std::atomic<int> known[64];
    const int fit = resident_clusters((const void*)kernel, known, cfg, C);
    if (fit > 0 && fit < most) most = fit;
    p.err = device_error_word();
  }
  const int grid = (int)(need < most ? need : most);
  p.width = C > 1 ? round_up(ceil_div(p.cols, C), VEC) : p.cols;
  cfg.gridDim = (unsigned)(grid * C);
  PL_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  count_launch();
  return p.part ? param_launch(p.part, grid, p.cols, dw1, dw2, st) : PL_OK;
}
// The smallest group of threads whose registers hold a row. Forward with 16 bf16 values per thread (65,536 x 2,048: 234 us, with
// 8 282), backward with 8, since it has six rows' worth of values in flight (16: 482 -> 882 us, spills); more forward beyond
// a block of 512 threads. Backward a row of more than 2,048 columns goes to a cluster, whose blocks keep these 8 (bf16 with
// gate, 268 MB per matrix: 4,096 columns in a block of 512 threads 487 us, in two of 256 452; 8,192 with 16 values per thread
// 649, two blocks 485; 16,384 1,490, four blocks 557). Without a gate the next row's load is on its way during the
// first fold already, and one block is better at 4,096 columns (290 us, two blocks 316; f32 244, 304).
// Forward, beyond 8,192 columns, a block of 1,024 threads has 64 registers for each: bf16 rows (spills of 208 bytes) and f32 rows
// without a gate still gain by it (8,192 x 16,384: 342 us, the walk below 468; f32 501, 574). f32 rows with a gate and
// rows without 16-byte loads do not, and are walked (604 bytes: 835 us, walked 683; 8,192 x 16,383 with gate bf16 641, 505, f32
// 1,888, 708).
#define PL_PICK_FWD(CALL)                  \
  if constexpr (sizeof(T) == 2) {          \
    if (cols <= 256) CALL(8, 32, 1);       \
    if (cols <= 512) CALL(8, 32, 2);       \
    if (cols <= 1024) CALL(8, 64, 2);      \
    if (cols <= 2048) CALL(8, 128, 2);     \
    if (cols <= 4096) CALL(8, 256, 2);     \
    if (cols <= 8192) CALL(8, 512, 2);     \
    if (cols <= 16384) CALL(8, 1024, 2);   \
  } else {                                 \
    PL_PICK_F32(CALL)                      \
  }
#define PL_PICK_BWD(CALL)                  \
  if constexpr (sizeof(T) == 2) {          \
    if (cols <= 256) CALL(8, 32, 1, 1);    \
    if (cols <= 512) CALL(8, 64, 1, 1);    \
    if (cols <= 1024) CALL(8, 128, 1, 1);  \
    if (cols <= 2048) CALL(8, 256, 1, 1);  \
    PL_PICK_CLUSTER(CALL, 8, 1)            \
  } else {                                 \
    if (cols <= 128) CALL(4, 32, 1, 1);    \
    if (cols <= 256) CALL(4, 32, 2, 1);    \
    if (cols <= 512) CALL(4, 64, 2, 1);    \
    if (cols <= 1024) CALL(4, 128, 2, 1);  \
    if (cols <= 2048) CALL(4, 256, 2, 1);  \
    PL_PICK_CLUSTER(CALL, 4, 2)            \
  }
#define PL_PICK_BWD_SINGLE(CALL)           \
  if (cols <= 128) CALL(1, 32, 4, 1);      \
  if (cols <= 512) CALL(1, 64, 8, 1);      \
  if (cols <= 1024) CALL(1, 128, 8, 1);    \
  if (cols <= 2048) CALL(1, 256, 8, 1);    \
  PL_PICK_CLUSTER(CALL, 1, 8)
#define PL_PICK_CLUSTER(CALL, VEC, K)                                                     \
  if (cols <= 4096 && !p.gate) return bwd_launch<T, VEC, 512, K, 1, false>(p, dw1, dw2, st); \
  if (cols <= 4096) return bwd_launch<T, VEC, 256, K, 2, true>(p, dw1, dw2, st);             \
  if (cols <= 8192) CALL(VEC, 512, K, 2);                                                 \
  if (cols <= 16384) CALL(VEC, 512, K, 4);
#define PL_PICK_F32(CALL)                  \
  if (cols <= 128) CALL(4, 32, 1);         \
  if (cols <= 256) CALL(4, 32, 2);         \
  if (cols <= 512) CALL(4, 64, 2);         \
  if (cols <= 1024) CALL(4, 128, 2);       \
  if (cols <= 2048) CALL(4, 256, 2);       \
  if (cols <= 4096) CALL(4, 512, 2);       \
  if (cols <= 8192) CALL(4, 512, 4);       \
  if (cols <= 16384 && !p.gate) return fwd_launch<T, 4, 1024, 4, false>(p, st);
#define PL_PICK_SINGLE(CALL)               \
  if (cols <= 128) CALL(1, 32, 4);         \
  if (cols <= 512) CALL(1, 64, 8);         \
  if (cols <= 1024) CALL(1, 128, 8);       \
  if (cols <= 2048) CALL(1, 256, 8);       \
  if (cols <= 4096) CALL(1, 512, 8);       \
  if (cols <= 8192) CALL(1, 512, 16);

static bool aligned16(const void* p) { return !p || ((uintptr_t)p & 15) == 0; }

template <typename T>
static int fwd_pick(const BlockArgs<T>& p, cudaStream_t st) {
  const long cols = p.cols;
  const bool vec = vec_ok(p.x, p.ldx, sizeof(T)) && vec_ok(p.branch, p.ldb, sizeof(T)) &&
                   (!p.gate || vec_ok(p.gate, p.ldg, sizeof(T))) && vec_ok(p.r, p.ldr, sizeof(T)) &&
                   vec_ok(p.y, p.ldy, sizeof(T)) && aligned16(p.w1) && aligned16(p.w2) &&
                   (cols * sizeof(T)) % 16 == 0;
#define PL_FWD(VEC, TPR, K) return fwd_launch<T, VEC, TPR, K>(p, st)
  if (vec) {
    PL_PICK_FWD(PL_FWD)
  } else {
    PL_PICK_SINGLE(PL_FWD)
  }
#undef PL_FWD
  PL_CUDA(launch_early(block_fwd_wide_kernel<T>, (unsigned)p.rows, 512, 0, st, p));
  count_launch();
  return PL_OK;
}
template <typename T>
static int bwd_pick(BlockGradArgs<T>& p, float* dw1, float* dw2, float* ws, cudaStream_t st) {
  const long cols = p.cols;
  p.part = (dw1 || dw2) ? ws : nullptr;
  const bool vec = vec_ok(p.dy, p.lddy, sizeof(T)) && vec_ok(p.branch, p.ldb, sizeof(T)) && vec_ok(p.r, p.ldr, sizeof(T)) &&
                   (!p.dr || vec_ok(p.dr, p.lddr, sizeof(T))) && vec_ok(p.dx, p.lddx, sizeof(T)) &&
                   vec_ok(p.db, p.lddb, sizeof(T)) &&
                   (!p.gate || (vec_ok(p.gate, p.ldg, sizeof(T)) && vec_ok(p.dg, p.lddg, sizeof(T)))) &&
                   aligned16(p.w1) && aligned16(p.w2) && (cols * sizeof(T)) % 16 == 0;
#define PL_BWD(VEC, TPR, K, C)                                                  \
  return p.gate ? bwd_launch<T, VEC, TPR, K, C, true>(p, dw1, dw2, st)         \
                : bwd_launch<T, VEC, TPR, K, C, false>(p, dw1, dw2, st)
  if (vec) {
    PL_PICK_BWD(PL_BWD)
  } else {
    PL_PICK_BWD_SINGLE(PL_BWD)
  }
#undef PL_BWD
  const int slices = (int)(p.rows < kWideSlices ? p.rows : kWideSlices);
  float* mean = p.part ? p.part + (long)slices * 2 * cols : nullptr;
  PL_CUDA(launch_early(block_bwd_wide_kernel<T>, (unsigned)p.rows, 512, 0, st, p, mean));
  count_launch();
  if (!p.part) return PL_OK;
  PL_CUDA(launch_early(block_bwd_wide_param_kernel<T>, dim3((unsigned)ceil_div(cols, 256), slices), 256, 0, st, p,
                       (const float*)mean));
  count_launch();
  return param_launch(p.part, slices, cols, dw1, dw2, st);
}
#undef PL_PICK_FWD
#undef PL_PICK_BWD
#undef PL_PICK_BWD_SINGLE
#undef PL_PICK_CLUSTER
#undef PL_PICK_F32
#undef PL_PICK_SINGLE

template <typename T>
static int block_fwd(const void* x, size_t ldx, const void* branch, size_t ldb, const void* gate, size_t ldg,
                     const float* w1, const float* w2, double scale, double eps, uint8_t post, size_t rows, size_t cols,
                     void* r, size_t ldr, void* y, size_t ldy, float* rstd_b, float* rstd, cudaStream_t st) {
  const BlockArgs<T> p = {(const T*)x, (const T*)branch, (const T*)gate, (long)ldx, (long)ldb, (long)ldg, w1, w2,
                          (float)scale, (float)eps, (long)rows, (long)cols, (T*)r, (T*)y, (long)ldr, (long)ldy,
                          post ? rstd_b : nullptr, rstd};
  return fwd_pick<T>(p, st);
}
template <typename T>
static int block_bwd(const void* dr, size_t lddr, const void* dy, size_t lddy, const void* branch, size_t ldb,
                     const void* gate, size_t ldg, const void* r, size_t ldr, const float* rstd_b, const float* rstd,
                     const float* w1, const float* w2, double scale, size_t rows, size_t cols, void* dx, size_t lddx,
                     void* db, size_t lddb, void* dg, size_t lddg, float* dw1, float* dw2, void* ws, cudaStream_t st) {
  BlockGradArgs<T> p = {(const T*)dr, (const T*)dy, (const T*)branch, (const T*)gate, (const T*)r, (long)lddr, (long)lddy,
                        (long)ldb, (long)ldg, (long)ldr, rstd_b, rstd, w1, w2, (float)scale, (long)rows, (long)cols,
                        (T*)dx, (T*)db, (T*)dg, (long)lddx, (long)lddb, (long)lddg, nullptr};
  return bwd_pick<T>(p, dw1, dw2, (float*)ws, st);
}

}  // namespace pl

extern "C" {

int pl_block_norm_dev(const void* x, size_t ldx, const void* branch, size_t ldb, const void* gate, size_t ldg,
                      const float* w_branch, const float* w, double scale, double eps, uint8_t post, size_t rows,
                      size_t cols, uint8_t bf16, void* r, size_t ldr, void* y, size_t ldy, float* rstd_branch,
                      float* rstd, void* stream) {
  using namespace pl;
  const char* me = "pl_block_norm_dev";
  PL_REQUIRE(cols > 0, PL_ERR_INVALID, "%s: rows of no columns", me);
  PL_REQUIRE(rows <= 0x7fffffffu && cols <= 0x7fffffffu, PL_ERR_INVALID, "%s: %zu x %zu is too large", me, rows, cols);
  PL_REQUIRE(ldx >= cols && ldb >= cols && (!gate || ldg >= cols) && ldr >= cols && ldy >= cols, PL_ERR_INVALID,
             "%s: a row stride is below %zu columns", me, cols);
  PL_REQUIRE(eps >= 0.0, PL_ERR_INVALID, "%s: eps = %g", me, eps);
  if (rows == 0) return PL_OK;
  PL_REQUIRE(x && branch && r && y && rstd && (!post || rstd_branch), PL_ERR_INVALID, "%s: NULL matrix or statistics", me);
  int rc = require_device();
  if (rc) return rc;
  return (bf16 ? block_fwd<__nv_bfloat16> : block_fwd<float>)(x, ldx, branch, ldb, gate, ldg, w_branch, w, scale, eps, post,
                                                              rows, cols, r, ldr, y, ldy, rstd_branch, rstd,
                                                              (cudaStream_t)stream);
}

size_t pl_block_norm_grad_ws(size_t rows, size_t cols) {
  const size_t most = (long)cols > pl::kBlockMost ? (size_t)pl::kWideSlices : (size_t)pl::kNormParts;
  const size_t parts = rows < most ? rows : most;
  return ((parts ? parts : 1) * 2 * cols + ((long)cols > pl::kBlockMost ? rows : 0)) * sizeof(float);
}

int pl_block_norm_grad_dev(const void* dr, size_t lddr, const void* dy, size_t lddy, const void* branch, size_t ldb,
                           const void* gate, size_t ldg, const void* r, size_t ldr, const float* rstd_branch,
                           const float* rstd, const float* w_branch, const float* w, double scale, size_t rows,
                           size_t cols, uint8_t bf16, void* dx, size_t lddx, void* dbranch, size_t lddb, void* dgate,
                           size_t lddg, float* dw_branch, float* dw, void* ws, size_t ws_bytes, void* stream) {
  using namespace pl;
  const char* me = "pl_block_norm_grad_dev";
  PL_REQUIRE(cols > 0, PL_ERR_INVALID, "%s: rows of no columns", me);
  PL_REQUIRE(rows <= 0x7fffffffu && cols <= 0x7fffffffu, PL_ERR_INVALID, "%s: %zu x %zu is too large", me, rows, cols);
  PL_REQUIRE((!dr || lddr >= cols) && lddy >= cols && ldb >= cols && (!gate || (ldg >= cols && lddg >= cols)) &&
                 ldr >= cols && lddx >= cols && lddb >= cols,
             PL_ERR_INVALID, "%s: a row stride is below %zu columns", me, cols);
  int rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (dw_branch) PL_CUDA(cudaMemsetAsync(dw_branch, 0, cols * 4, st));
    if (dw) PL_CUDA(cudaMemsetAsync(dw, 0, cols * 4, st));
    return PL_OK;
  }
  PL_REQUIRE(dy && branch && r && rstd && dx && dbranch && (!gate || dgate), PL_ERR_INVALID,
             "%s: NULL matrix or statistics", me);
  if (dw_branch || dw)
    PL_REQUIRE(ws && ((uintptr_t)ws & 3) == 0 && ws_bytes >= pl_block_norm_grad_ws(rows, cols), PL_ERR_INVALID,
               "%s: %zu bytes of workspace, %zu needed", me, ws ? ws_bytes : (size_t)0, pl_block_norm_grad_ws(rows, cols));
  return (bf16 ? block_bwd<__nv_bfloat16> : block_bwd<float>)(dr, lddr, dy, lddy, branch, ldb, gate, ldg, r, ldr,
                                                              rstd_branch, rstd, w_branch, w, scale, rows, cols, dx, lddx,
                                                              dbranch, lddb, dgate, lddg, dw_branch, dw, ws, st);
}

}  // extern "C"
