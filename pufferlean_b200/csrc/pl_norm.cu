// Layer norm over the rows of a matrix, forward and backward (f32 or bf16 rows; statistics, weight, bias and
// every sum in f32).
//
//   forward   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), y = (x - m) r w + b
//   backward  xh = (x - m) r, g = dy w, dx = r (g - mean g - xh mean(g xh)), dw = sum_rows dy xh, db = sum_rows dy
//
// Both directions are bound by HBM: 2 (forward) or 3 (backward) passes over rows x cols values and nothing else
// of that size. So a row is read once and stays in registers: TPR threads own a row, thread t its columns
// (k TPR + t) VEC + j, k < K, j < VEC, with 16-byte loads where base, row stride and width allow them and single
// values otherwise. The variance is taken about the mean (a second pass over the registers, not over memory).
//
// Measured, us and share of a copy's 6,449 GB/s: 65,536 x 2,048 bf16 forward 93 (90 %), backward 149 (84 %); 65,536 x
// 1,024 f32 forward 88 (95 %). Less is reached where values go singly (65,536 x 1,003 bf16: 74 and 114, 55 and 54 %) and
// in rows of more than 8,192 columns: up to 16,384 a block of 1,024 threads has 64 registers each and spills (forward
// 48 to 112 bytes a thread, backward 344 to 544; 8,192 x 16,384 bf16: 161 and 319, 52 and 39 %; f32: 198 and 602, 84 and
// 41 %), and beyond that rows are read again from L2, value by value (4,096 x 20,000 bf16: 127 and 283, 40 and 27 %).
#include "pl_rows.cuh"
#include "pl_runtime.h"

namespace pl {

// A block walks the rows, RB of them per group at a time, their sums folded in one butterfly and the weights kept in
// registers (read again per row they cost twice the row's own L1 traffic: 65,536 x 2,048 bf16 took 135 us that way).
// The next rows are loaded one step ahead; bulk copies into a ring of shared memory instead were no faster (107
// against 95 us: what bounds the kernel then is the folds' latency, not the loads').
template <typename T, int VEC, int TPR, int K, int RB>
__global__ void __launch_bounds__(norm_threads(TPR), norm_blocks(TPR))
    norm_fwd_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w, const float* __restrict__ b,
                    long rows, int cols, float eps, T* __restrict__ y, long ldy, float* __restrict__ mean,
                    float* __restrict__ rstd) {
  grid_wait();
  grid_next();
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR, LV = 32 / RB;
  __shared__ float scr[2][RB][32];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inv = 1.f / (float)cols;
  const long step = (long)gridDim.x * G * RB, base0 = (long)blockIdx.x * G * RB;
  Vec<VEC> wv[K], bv[K];
  bool in_row[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int c = (k * TPR + t) * VEC;
    in_row[k] = c < cols;
    wv[k] = vall<VEC>(1.f);
    bv[k] = vall<VEC>(0.f);
    if (w && in_row[k]) load_param<VEC>(w, c, wv[k].v);
    if (b && in_row[k]) load_param<VEC>(b, c, bv[k].v);
  }
  Pack<T, VEC> nx[RB][K];
  auto load = [&](long r0) {  // what lies outside the matrix reads as zero
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (r0 + i < rows && in_row[k])
          nx[i][k].load(x + (r0 + i) * ldx + (k * TPR + t) * VEC);
        else
          nx[i][k] = narrow<T, VEC>(vall<VEC>(0.f));
      }
  };
  load(base0 + g * RB);
  for (long base = base0; base < rows; base += step) {
    const long r0 = base + (long)g * RB;
    Vec<VEC> f[RB][K];
    float s[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) {
      Vec<VEC> a = vall<VEC>(0.f);
#pragma unroll
      for (int k = 0; k < K; k++) {
        f[i][k] = widen<T, VEC>(nx[i][k]);
        a = vadd(a, f[i][k]);
      }
      s[i] = vsum(a);
    }
    if (base + step < rows) load(r0 + step);
    float v = group_sum_n<TPR, RB>(s, scr[0], lane, warp) * inv;
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const float m = __shfl_sync(0xffffffffu, v, i * LV);
      if (t == 0 && r0 + i < rows) mean[r0 + i] = m;
      Vec<VEC> a = vall<VEC>(0.f);
#pragma unroll
      for (int k = 0; k < K; k++) {
        f[i][k] = vadd(f[i][k], vall<VEC>(-m));
        if (in_row[k]) a = vfma(f[i][k], f[i][k], a);
      }
      s[i] = vsum(a);
    }
    v = group_sum_n<TPR, RB>(s, scr[1], lane, warp);  // its barrier also ends the reads of scr[0]
    v = 1.f / sqrtf(v * inv + eps);
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const float r = __shfl_sync(0xffffffffu, v, i * LV);
      if (r0 + i >= rows) break;
      if (t == 0) rstd[r0 + i] = r;
#pragma unroll
      for (int k = 0; k < K; k++)
        if (in_row[k])
          narrow<T, VEC>(vfma(vmul(f[i][k], vall<VEC>(r)), wv[k], bv[k])).store(y + (r0 + i) * ldy + (k * TPR + t) * VEC);
    }
  }
}

// Rows too wide for the registers: one block per row, the row read three times (its second and third reads hit
// L2).
template <typename T>
__global__ void __launch_bounds__(512)
    norm_fwd_wide_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w, const float* __restrict__ b,
                         long rows, long cols, float eps, T* __restrict__ y, long ldy, float* __restrict__ mean,
                         float* __restrict__ rstd) {
  grid_wait();
  grid_next();
  __shared__ float scr[2][32];
  const long row = blockIdx.x;
  const T* xr = x + row * ldx;
  const float inv = 1.f / (float)cols;
  float s = 0.f;
  for (long c = threadIdx.x; c < cols; c += 512) s += to_f(xr[c]);
  const float m = group_sum<512>(s, scr[0]) * inv;
  s = 0.f;
  for (long c = threadIdx.x; c < cols; c += 512) {
    const float d = to_f(xr[c]) - m;
    s = __fmaf_rn(d, d, s);
  }
  const float r = 1.f / sqrtf(group_sum<512>(s, scr[1]) * inv + eps);
  if (threadIdx.x == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
  for (long c = threadIdx.x; c < cols; c += 512) {
    float v = (to_f(xr[c]) - m) * r;
    if (w) v *= w[c];
    if (b) v += b[c];
    y[row * ldy + c] = from_f<T>(v);
  }
}

// ---------------------------------------------------------------------------------------------- backward
// A block walks the rows with RB of them per group in flight: the two row sums of RB rows are folded in one
// butterfly, and each thread adds its columns of dy xh and dy to registers over all of its block's rows. The
// blocks' column sums go to `part` ([grid][2][cols]) and are added in block order by norm_param_kernel.
// Wide rows leave few registers per thread: RB falls, and the weight is read again (from L1) for each row.
template <typename T, int VEC, int TPR, int K, int RB>
__global__ void __launch_bounds__(norm_threads(TPR), norm_blocks(TPR))
    norm_bwd_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                    const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                    long rows, int cols, T* __restrict__ dx, long lddx, float* __restrict__ part) {
  grid_wait();
  grid_next();
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR, E = VEC * K;
  constexpr int NV = 2 * RB, LV = 32 / NV;  // values of an iteration, lanes that hold one of them
  constexpr bool KEEP_W = TPR < 1024;
  __shared__ float scr[2][NV][32];  // [iteration parity][value][warp]
  extern __shared__ float fold[];   // [G][2][TPR * E] (G > 1)
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inv = 1.f / (float)cols;
  const long step = (long)gridDim.x * G * RB, base0 = (long)blockIdx.x * G * RB;
  Vec<VEC> wv[K], dw[K], db[K];
  bool in_row[K];
  auto load_w = [&](int k) {
    wv[k] = vall<VEC>(1.f);
    const int c = (k * TPR + t) * VEC;
    if (w && c < cols) load_param<VEC>(w, c, wv[k].v);
  };
#pragma unroll
  for (int k = 0; k < K; k++) in_row[k] = (k * TPR + t) * VEC < cols;
#pragma unroll
  for (int k = 0; k < K; k++) {
    dw[k] = db[k] = vall<VEC>(0.f);
    if (KEEP_W) load_w(k);
  }
  Pack<T, VEC> xn[RB][K], dn[RB][K];
  float mn[RB], rn[RB];
  auto load = [&](long r0) {  // what lies outside the matrix: dy = 0 keeps it out of every sum
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const bool ok = r0 + i < rows;
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (ok && in_row[k]) {
          xn[i][k].load(x + (r0 + i) * ldx + (k * TPR + t) * VEC);
          dn[i][k].load(dy + (r0 + i) * lddy + (k * TPR + t) * VEC);
        } else {
          xn[i][k] = dn[i][k] = narrow<T, VEC>(vall<VEC>(0.f));
        }
      }
      mn[i] = ok ? __ldg(mean + r0 + i) : 0.f;
      rn[i] = ok ? __ldg(rstd + r0 + i) : 0.f;
    }
  };
  load(base0 + g * RB);
  int parity = 0;
  for (long base = base0; base < rows; base += step, parity ^= 1) {
    const long r0 = base + (long)g * RB;
    Vec<VEC> xh[RB][K], gg[RB][K];
    float r[RB], s[NV];
#pragma unroll
    for (int i = 0; i < RB; i++) {
      r[i] = rn[i];
      Vec<VEC> s1 = vall<VEC>(0.f), s2 = vall<VEC>(0.f);
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (!KEEP_W) load_w(k);
        const Vec<VEC> d = widen<T, VEC>(dn[i][k]);
        xh[i][k] = vmul(vadd(widen<T, VEC>(xn[i][k]), vall<VEC>(-mn[i])), vall<VEC>(r[i]));
        gg[i][k] = vmul(d, wv[k]);
        s1 = vadd(s1, gg[i][k]);
        s2 = vfma(gg[i][k], xh[i][k], s2);
        dw[k] = vfma(d, xh[i][k], dw[k]);
        db[k] = vadd(db[k], d);
      }
      s[2 * i] = vsum(s1);
      s[2 * i + 1] = vsum(s2);
    }
    if (base + step < rows) load(r0 + step);
    const float v = -inv * group_sum_n<TPR, NV>(s, scr[parity], lane, warp);  // the other parity's barrier ended its reads
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const Vec<VEC> a1 = vall<VEC>(__shfl_sync(0xffffffffu, v, 2 * i * LV));        // - mean of g
      const Vec<VEC> a2 = vall<VEC>(__shfl_sync(0xffffffffu, v, (2 * i + 1) * LV));  // - mean of g xh
      if (r0 + i >= rows) break;
#pragma unroll
      for (int k = 0; k < K; k++)
        if (in_row[k])
          narrow<T, VEC>(vmul(vfma(xh[i][k], a2, vadd(gg[i][k], a1)), vall<VEC>(r[i])))
              .store(dx + (r0 + i) * lddx + (k * TPR + t) * VEC);
    }
  }
  if (!part) return;
  float* pw = part + (long)blockIdx.x * 2 * cols;
  if constexpr (G > 1) {
    constexpr int W = TPR * E;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const int c = (k * TPR + t) * VEC + j;
        fold[(g * 2) * W + c] = dw[k].v[j];
        fold[(g * 2 + 1) * W + c] = db[k].v[j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += THREADS) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < G; q++) {
        a += fold[(q * 2) * W + c];
        b += fold[(q * 2 + 1) * W + c];
      }
      pw[c] = a;
      pw[cols + c] = b;
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const int c = (k * TPR + t) * VEC + j;
        if (c < cols) {
          pw[c] = dw[k].v[j];
          pw[cols + c] = db[k].v[j];
        }
      }
  }
}

// dw[c] = sum_p part[p][0][c], db[c] = sum_p part[p][1][c]: 32 columns per block, 32 slices of the parts, both
// folded in a fixed order.
__global__ void __launch_bounds__(1024)
    norm_param_kernel(const float* __restrict__ part, int parts, long cols, float* __restrict__ dw,
                      float* __restrict__ db) {
  grid_wait();
  grid_next();
  __shared__ float scr[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long c = (long)blockIdx.x * 32 + lane;
  const float* p = part + (blockIdx.y ? cols : 0);
  float s = 0.f;
  if (c < cols) {
#pragma unroll 10
    for (int q = slice; q < parts; q += 32) s += __ldg(p + (long)q * 2 * cols + c);
  }
  scr[slice][lane] = s;
  __syncthreads();
  s = warp_sum(scr[lane][slice]);  // warp `slice` folds column `slice` of the block
  const long o = (long)blockIdx.x * 32 + slice;
  float* out = blockIdx.y ? db : dw;
  if (lane == 0 && o < cols && out) out[o] = s;
}

// Rows too wide for the registers. dx: one block per row, both inputs read twice.
template <typename T>
__global__ void __launch_bounds__(512)
    norm_bwd_wide_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                         const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                         long rows, long cols, T* __restrict__ dx, long lddx) {
  grid_wait();
  grid_next();
  __shared__ float scr[2][32];
  const long row = blockIdx.x;
  const float m = mean[row], r = rstd[row], inv = 1.f / (float)cols;
  const T *xr = x + row * ldx, *dr = dy + row * lddy;
  float s1 = 0.f, s2 = 0.f;
  for (long c = threadIdx.x; c < cols; c += 512) {
    const float g = to_f(dr[c]) * (w ? w[c] : 1.f);
    s1 += g;
    s2 = __fmaf_rn(g, (to_f(xr[c]) - m) * r, s2);
  }
  const float a1 = group_sum<512>(s1, scr[0]) * inv, a2 = group_sum<512>(s2, scr[1]) * inv;
  for (long c = threadIdx.x; c < cols; c += 512) {
    const float g = to_f(dr[c]) * (w ? w[c] : 1.f);
    dx[row * lddx + c] = from_f<T>((g - a1 - (to_f(xr[c]) - m) * r * a2) * r);
  }
}
// dw, db: one thread per column and slice of the rows, [gridDim.y][2][cols] parts.
template <typename T>
__global__ void __launch_bounds__(256)
    norm_bwd_wide_param_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                               const float* __restrict__ mean, const float* __restrict__ rstd, long rows, long cols,
                               float* __restrict__ part) {
  grid_wait();
  grid_next();
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float a = 0.f, b = 0.f;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = to_f(dy[r * lddy + c]);
    a = __fmaf_rn(d, (to_f(x[r * ldx + c]) - mean[r]) * rstd[r], a);
    b += d;
  }
  float* p = part + (long)blockIdx.y * 2 * cols;
  p[c] = a;
  p[cols + c] = b;
}

// ---------------------------------------------------------------------------------------------- host side
template <typename T, int VEC, int TPR, int K, int RB>
static int fwd_launch(const void* x, long ldx, const float* w, const float* b, long rows, int cols, float eps, void* y,
                      long ldy, float* mean, float* rstd, cudaStream_t st) {
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  const long need = ceil_div(rows, (long)G * RB), most = (long)kNormSms * norm_blocks(TPR);
  // few rows: one per group, so that more SMs have some (latency); many: RB at a time
  if constexpr (RB > 1)
    if (need < most / 2) return fwd_launch<T, VEC, TPR, K, 1>(x, ldx, w, b, rows, cols, eps, y, ldy, mean, rstd, st);
  PL_CUDA(launch_early(norm_fwd_kernel<T, VEC, TPR, K, RB>, (unsigned)(need < most ? need : most), THREADS, 0, st,
                        (const T*)x, ldx, w, b, rows, cols, eps, (T*)y, ldy, mean, rstd));
  count_launch();
  return PL_OK;
}

template <typename T>
static int fwd_pick(const void* x, long ldx, const float* w, const float* b, long rows, long cols, float eps, void* y,
                    long ldy, float* mean, float* rstd, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = vec_ok(x, ldx, sizeof(T)) && vec_ok(y, ldy, sizeof(T)) && cols % V == 0 &&
                   (!w || ((uintptr_t)w & 15) == 0) && (!b || ((uintptr_t)b & 15) == 0);
#define PL_FWD(VEC, TPR, K, RB)    \
  if (cols <= (long)VEC * TPR * K) \
    return fwd_launch<T, VEC, TPR, K, RB>(x, ldx, w, b, rows, (int)cols, eps, y, ldy, mean, rstd, st);
  if (vec) {
    if constexpr (V == 8) {  // bf16: 16 values per thread
      PL_FWD(V, 32, 1, 4)
      PL_FWD(V, 32, 2, 2)
      PL_FWD(V, 64, 2, 2)
      PL_FWD(V, 128, 2, 2)
      PL_FWD(V, 256, 2, 2)
      PL_FWD(V, 512, 2, 2)
      PL_FWD(V, 1024, 2, 1)
    } else {
      PL_FWD(V, 32, 1, 4)
      PL_FWD(V, 64, 1, 4)
      PL_FWD(V, 128, 1, 4)
      PL_FWD(V, 256, 1, 4)
      PL_FWD(V, 512, 1, 4)
      PL_FWD(V, 512, 2, 2)
      PL_FWD(V, 1024, 2, 1)
      PL_FWD(V, 1024, 4, 1)
    }
  } else {
    PL_FWD(1, 32, 4, 4)
    PL_FWD(1, 64, 8, 2)
    PL_FWD(1, 128, 8, 2)
    PL_FWD(1, 256, 8, 2)
    PL_FWD(1, 512, 8, 1)
    PL_FWD(1, 1024, 8, 1)
    PL_FWD(1, 1024, 16, 1)
  }
#undef PL_FWD
  PL_CUDA(launch_early(norm_fwd_wide_kernel<T>, (unsigned)rows, 512, 0, st, (const T*)x, ldx, w, b, rows, cols, eps,
                       (T*)y, ldy, mean, rstd));
  count_launch();
  return PL_OK;
}

int param_launch(const float* part, int parts, long cols, float* dw, float* db, cudaStream_t st) {
  PL_CUDA(launch_early(norm_param_kernel, dim3((unsigned)ceil_div(cols, 32), 2), 1024, 0, st, part, parts, cols, dw,
                       db));
  count_launch();
  return PL_OK;
}

template <typename T, int VEC, int TPR, int K, int RB>
static int bwd_launch(const void* dy, long lddy, const void* x, long ldx, const float* w, const float* mean,
                      const float* rstd, long rows, int cols, void* dx, long lddx, float* dw, float* db, float* part,
                      cudaStream_t st) {
  constexpr int THREADS = norm_threads(TPR), G = THREADS / TPR;
  constexpr size_t FOLD = G > 1 ? (size_t)G * 2 * TPR * VEC * K * 4 : 0;
  const long need = ceil_div(rows, (long)G * RB), most = (long)kNormSms * norm_blocks(TPR);
  if constexpr (RB > 1)
    if (need < most / 2)
      return bwd_launch<T, VEC, TPR, K, 1>(dy, lddy, x, ldx, w, mean, rstd, rows, cols, dx, lddx, dw, db, part, st);
  const int grid = (int)(need < most ? need : most);
  static_assert(FOLD <= 48 * 1024, "column sums of the groups");
  PL_CUDA(launch_early(norm_bwd_kernel<T, VEC, TPR, K, RB>, grid, THREADS, FOLD, st, (const T*)dy, lddy, (const T*)x,
                       ldx, w, mean, rstd, rows, cols, (T*)dx, lddx, (dw || db) ? part : nullptr));
  count_launch();
  return (dw || db) ? param_launch(part, grid, cols, dw, db, st) : PL_OK;
}

template <typename T>
static int bwd_pick(const void* dy, long lddy, const void* x, long ldx, const float* w, const float* mean,
                    const float* rstd, long rows, long cols, void* dx, long lddx, float* dw, float* db, float* part,
                    cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = vec_ok(x, ldx, sizeof(T)) && vec_ok(dy, lddy, sizeof(T)) && vec_ok(dx, lddx, sizeof(T)) &&
                   cols % V == 0 && (!w || ((uintptr_t)w & 15) == 0);
#define PL_BWD(VEC, TPR, K, RB)    \
  if (cols <= (long)VEC * TPR * K) \
    return bwd_launch<T, VEC, TPR, K, RB>(dy, lddy, x, ldx, w, mean, rstd, rows, (int)cols, dx, lddx, dw, db, part, st);
  if (vec) {
    if constexpr (V == 8) {
      PL_BWD(V, 32, 1, 2)
      PL_BWD(V, 32, 2, 1)
      PL_BWD(V, 64, 2, 1)
      PL_BWD(V, 128, 2, 1)
      PL_BWD(V, 256, 2, 1)
      PL_BWD(V, 512, 2, 1)
      PL_BWD(V, 1024, 2, 1)
    } else {
      PL_BWD(V, 32, 1, 4)
      PL_BWD(V, 64, 1, 4)
      PL_BWD(V, 128, 1, 4)
      PL_BWD(V, 256, 1, 4)
      PL_BWD(V, 512, 1, 4)
      PL_BWD(V, 512, 2, 2)
      PL_BWD(V, 1024, 2, 1)
      PL_BWD(V, 1024, 4, 1)
    }
  } else {
    PL_BWD(1, 32, 4, 4)
    PL_BWD(1, 64, 8, 2)
    PL_BWD(1, 128, 8, 2)
    PL_BWD(1, 256, 8, 2)
    PL_BWD(1, 512, 8, 1)
    PL_BWD(1, 1024, 8, 1)
    PL_BWD(1, 1024, 16, 1)
  }
#undef PL_BWD
  PL_CUDA(launch_early(norm_bwd_wide_kernel<T>, (unsigned)rows, 512, 0, st, (const T*)dy, lddy, (const T*)x, ldx, w,
                       mean, rstd, rows, cols, (T*)dx, lddx));
  count_launch();
  if (!dw && !db) return PL_OK;
  const int slices = (int)(rows < 64 ? rows : 64);
  PL_CUDA(launch_early(norm_bwd_wide_param_kernel<T>, dim3((unsigned)ceil_div(cols, 256), slices), 256, 0, st,
                        (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, rows, cols, part));
  count_launch();
  return param_launch(part, slices, cols, dw, db, st);
}

}  // namespace pl

extern "C" {

int pl_layernorm_dev(const void* x, size_t ldx, const float* w, const float* b, size_t rows, size_t cols, double eps,
                     uint8_t bf16, void* y, size_t ldy, float* mean, float* rstd, void* stream) {
  using namespace pl;
  PL_REQUIRE(cols > 0, PL_ERR_INVALID, "pl_layernorm_dev: rows of no columns");
  PL_REQUIRE(rows <= 0x7fffffffu && cols <= 0x7fffffffu, PL_ERR_INVALID, "pl_layernorm_dev: %zu x %zu is too large", rows,
             cols);
  PL_REQUIRE(ldx >= cols && ldy >= cols, PL_ERR_INVALID, "pl_layernorm_dev: row strides %zu, %zu below %zu columns", ldx,
             ldy, cols);
  PL_REQUIRE(eps >= 0.0, PL_ERR_INVALID, "pl_layernorm_dev: eps = %g", eps);
  if (rows == 0) return PL_OK;
  PL_REQUIRE(x && y && mean && rstd, PL_ERR_INVALID, "pl_layernorm_dev: NULL matrix or statistics");
  int rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return bf16 ? fwd_pick<__nv_bfloat16>(x, (long)ldx, w, b, (long)rows, (long)cols, (float)eps, y, (long)ldy, mean, rstd, st)
              : fwd_pick<float>(x, (long)ldx, w, b, (long)rows, (long)cols, (float)eps, y, (long)ldy, mean, rstd, st);
}

size_t pl_layernorm_grad_ws(size_t rows, size_t cols) {
  const size_t parts = rows < (size_t)pl::kNormParts ? rows : (size_t)pl::kNormParts;
  return (parts ? parts : 1) * 2 * cols * sizeof(float);
}

int pl_layernorm_grad_dev(const void* dy, size_t lddy, const void* x, size_t ldx, const float* w, const float* mean,
                          const float* rstd, size_t rows, size_t cols, uint8_t bf16, void* dx, size_t lddx, float* dw,
                          float* db, void* ws, size_t ws_bytes, void* stream) {
  using namespace pl;
  PL_REQUIRE(cols > 0, PL_ERR_INVALID, "pl_layernorm_grad_dev: rows of no columns");
  PL_REQUIRE(rows <= 0x7fffffffu && cols <= 0x7fffffffu, PL_ERR_INVALID, "pl_layernorm_grad_dev: %zu x %zu is too large",
             rows, cols);
  PL_REQUIRE(ldx >= cols && lddy >= cols && lddx >= cols, PL_ERR_INVALID,
             "pl_layernorm_grad_dev: row strides %zu, %zu, %zu below %zu columns", lddy, ldx, lddx, cols);
  int rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (dw) PL_CUDA(cudaMemsetAsync(dw, 0, cols * 4, st));
    if (db) PL_CUDA(cudaMemsetAsync(db, 0, cols * 4, st));
    return PL_OK;
  }
  PL_REQUIRE(dy && x && mean && rstd && dx, PL_ERR_INVALID, "pl_layernorm_grad_dev: NULL matrix or statistics");
  if (dw || db)
    PL_REQUIRE(ws && ws_bytes >= pl_layernorm_grad_ws(rows, cols), PL_ERR_INVALID,
               "pl_layernorm_grad_dev: %zu bytes of workspace, %zu needed", ws ? ws_bytes : (size_t)0,
               pl_layernorm_grad_ws(rows, cols));
  return bf16 ? bwd_pick<__nv_bfloat16>(dy, (long)lddy, x, (long)ldx, w, mean, rstd, (long)rows, (long)cols, dx,
                                        (long)lddx, dw, db, (float*)ws, st)
              : bwd_pick<float>(dy, (long)lddy, x, (long)ldx, w, mean, rstd, (long)rows, (long)cols, dx, (long)lddx, dw,
                                db, (float*)ws, st);
}

}  // extern "C"
