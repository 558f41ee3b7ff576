// A large-vocabulary head and what it is trained with: softmax cross entropy against one target per row, and
// distillation from a teacher's top logits, forward and with gradients. The losses alone keep no logits; the gradients
// keep the softmax terms of a piece of the rows, 2 bytes each.
//
//   u = (x W^T + bias) / T          rows n < N, vocabulary v < V, hidden width D
//   lse_n = log sum_v exp u_nv      p_nk: the answer's probabilities (one entry of 1, or softmax(teacher / T))
//   loss_n = sum_k p_nk (log p_nk - u_n,id(n,k)) + lse_n
//   dz = scale_n / T (exp(u - lse) - sum_k p_nk onehot(id(n,k))),   dx = dz W,  dW = dz^T x,  dbias = sum_n dz
//
// Rows without an answer (a negative target, no entry present) are taken out before the products: a plan kernel
// lists the rows that count, the products' row extent is read from the device. One product gives the logits: its
// epilogue (pl_gemm.cuh, EPI_VOCAB) folds each row's 128 columns to (max, sum) and, when gradients are wanted,
// leaves 2^(u - max) in f16 for a piece of the rows. Once the rows' statistics are known these terms become dz in
// place (bf16, the one rounding of the gradient), and two more products give dx and dW. Three products of 2 N V D
// flops are also the least that the gradients need; recomputing the logits instead of keeping the terms would make it
// four.
//
// What bounds it: the three products run at the rate of the tensor cores under the power cap (16,384 x 131,072 x 2,048:
// 22.9 to 26.5 ms by board for 26.4 TFLOP; 18.8 ms at the 1,405 TFLOP/s that cuBLAS holds for seconds); the
// pass from terms to gradients at HBM's (2,048 x 131,072: 161 us for 1.07 GB); with few rows the reading of W and the
// writing of dW; with few rows of a small vocabulary the launches.
#include <cuda_fp16.h>

#include "../../include/pufferlean_b200_testing.h"
#include "pl_common.cuh"
#include "pl_gemm.cuh"
#include "pl_runtime.h"

namespace pl {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Which rows count: a target that is not negative (cross entropy), or `has` (distillation).
struct Answers {
  const int* target;
  const uint8_t* has;
};
__device__ __forceinline__ bool row_counts(const Answers& a, long row) {
  return a.target ? __ldg(a.target + row) >= 0 : (a.has ? __ldg(a.has + row) != 0 : true);
}
__device__ __forceinline__ long rows_here(const int* count, long off, long n) {
  return count ? min(n, max(0L, (long)*count - off)) : n;
}
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max_f(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The teacher's side of every row, one warp each: p = softmax(teacher / T) over the present entries (f32), entries
// that name one id added up in the first of them (the others become absent), and ent = sum_k p_k log2 p_k of the
// single entries. ids2, p [N][K]; a row without entries gets has = 0.
__global__ void __launch_bounds__(128)
    vocab_teacher_kernel(const int* __restrict__ ids, const float* __restrict__ teacher, long N, int K, float tscale,
                         int* __restrict__ ids2, float* __restrict__ p, float* __restrict__ ent,
                         uint8_t* __restrict__ has) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) uint8_t dyn_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long r = (long)blockIdx.x * 4 + warp;
  if (r >= N) return;
  const int K4 = (K + 3) / 4 * 4;
  int* id_s = reinterpret_cast<int*>(dyn_smem) + warp * 2 * K4;
  float* p_s = reinterpret_cast<float*>(id_s + K4);
  float top = -INFINITY;
  bool any = false;
  for (int k = lane; k < K4; k += 32) {
    int id = k < K ? ids[r * K + k] : -1;
    const float t = k < K ? teacher[r * K + k] : -INFINITY;
    if (t == -INFINITY) id = -1;
    id_s[k] = id;
    p_s[k] = t;
    if (id >= 0) {
      top = fmaxf(top, t);
      any = true;
    }
  }
  any = __any_sync(0xffffffffu, any);
  top = warp_max_f(top);
  float tot = 0.f;
  for (int k = lane; k < K; k += 32)
    if (id_s[k] >= 0) tot += exp2f((p_s[k] - top) * tscale);
  tot = warp_sum_f(tot);
  const float log_tot = log2f(tot);
  float e = 0.f;
  for (int k = lane; k < K4; k += 32) {
    float q = 0.f;
    if (id_s[k] >= 0) {
      const float l = (p_s[k] - top) * tscale - log_tot;
      q = exp2f(l);
      if (!(q == 0.f)) e = __fmaf_rn(q, l, e);
    }
    p_s[k] = q;
  }
  e = warp_sum_f(e);
  __syncwarp();
  for (int k = lane; k < K; k += 32) {
    const int id = id_s[k];
    float q = 0.f;
    bool first = id >= 0;
#pragma unroll 2
    for (int g = 0; g < K4; g += 4) {  // every entry of this id from k on; one before k makes it that one's
      const int4 i4 = *reinterpret_cast<const int4*>(id_s + g);
      const float4 p4 = *reinterpret_cast<const float4*>(p_s + g);
      if (i4.x == id) q += p4.x, first = first && g >= k;
      if (i4.y == id) q += p4.y, first = first && g + 1 >= k;
      if (i4.z == id) q += p4.z, first = first && g + 2 >= k;
      if (i4.w == id) q += p4.w, first = first && g + 3 >= k;
    }
    ids2[r * K + k] = first ? id : -1;
    p[r * K + k] = first ? q : 0.f;
  }
  if (lane == 0) {
    ent[r] = e;
    has[r] = any;
  }
}

// rows[0 .. *count) = the rows that count, in order; loss = lse = 0 for the others. One block, four rows to a thread.
__global__ void __launch_bounds__(1024)
    vocab_plan_kernel(Answers a, long N, int* __restrict__ rows, int* __restrict__ count, float* __restrict__ loss,
                      float* __restrict__ lse) {
  grid_wait();
  grid_next();
  __shared__ int warp_n[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (long r0 = 0; r0 < N; r0 += 4096) {
    const long r = r0 + 4 * threadIdx.x;
    bool in[4];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      in[j] = r + j < N && row_counts(a, r + j);
      mine += in[j];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    if (lane == 31) warp_n[warp] = upto;
    __syncthreads();
    int n = warp_n[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += t;
    }
    const int before = __shfl_sync(0xffffffffu, n, (warp + 31) & 31);
    int at = base + (warp ? before : 0) + upto - mine;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (in[j]) {
        rows[at++] = (int)(r + j);
      } else if (r + j < N) {
        loss[r + j] = 0.f;
        lse[r + j] = 0.f;
      }
    }
    base += __shfl_sync(0xffffffffu, n, 31);
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// Eight values at s, which need not be aligned: from the two 16-byte words that hold them. Reads the seven values
// before s and after s + 8 at most.
__device__ __forceinline__ uint4 load8_any(const __nv_bfloat16* s) {
  const uint32_t sh = (uint32_t)((uintptr_t)s & 15);
  const uint4* p = reinterpret_cast<const uint4*>((uintptr_t)s - sh);
  const uint4 a = p[0];
  if (sh == 0) return a;
  const uint4 b = p[1];
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const uint32_t q = sh >> 2, bits = (sh & 3) * 8;
  uint32_t u[5];
#pragma unroll
  for (int j = 0; j < 5; j++)
    u[j] = q == 0 ? w[j] : (q == 1 ? w[j + 1] : (q == 2 ? w[j + 2] : w[j + 3 < 8 ? j + 3 : 7]));
  return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits),
                    __funnelshift_r(u[2], u[3], bits), __funnelshift_r(u[3], u[4], bits));
}

// A warp's part of a row: values [c0, c0 + 1,024) of D, of any alignment on either side; zeros if not `in`. The middle
// goes 16 bytes to a lane, aligned where it is written.
__device__ __forceinline__ void copy_row(__nv_bfloat16* __restrict__ d, const __nv_bfloat16* __restrict__ s, long c0, long D,
                                         bool in, int lane) {
  const __nv_bfloat16 zero = __float2bfloat16_rn(0.f);
  const long c1 = min(D, c0 + 1024);
  const long head = min(c1, c0 + (long)((16 - ((uintptr_t)(d + c0) & 15)) & 15) / 2);  // first aligned value
  const bool same = (((uintptr_t)d ^ (uintptr_t)s) & 15) == 0;
  if (c0 + lane < head) d[c0 + lane] = in ? s[c0 + lane] : zero;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const long c = head + 256 * k + lane * 8;
    if (c + 8 <= c1) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (in) {
        if (same || (c >= 7 && c + 15 <= D)) {
          v = load8_any(s + c);
        } else {  // the row's ends, value by value
          __align__(16) __nv_bfloat16 t[8];
#pragma unroll
          for (int j = 0; j < 8; j++) t[j] = s[c + j];
          v = *reinterpret_cast<const uint4*>(t);
        }
      }
      *reinterpret_cast<uint4*>(d + c) = v;
    }
  }
  const long tail = head + (c1 - head) / 8 * 8 + lane;
  if (tail < c1) d[tail] = in ? s[tail] : zero;
}

// dst[i] = src[row i] for i < n (row i = rows[off + i] of the plan, or i itself without one; the row is zero where
// it does not count), rows up to the next multiple of 64 zeroed; with `again` the same once more that many rows below.
// One warp per row and 1,024 columns.
__global__ void __launch_bounds__(256)
    vocab_pack_kernel(const __nv_bfloat16* __restrict__ src, long ld, long D, Answers a, const int* __restrict__ rows,
                      const int* __restrict__ count, long off, long n, __nv_bfloat16* __restrict__ dst, long ldd,
                      long again) {
  grid_wait();
  grid_next();
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long have = rows_here(count, off, n);
  if (i >= (have + 63) / 64 * 64) return;
  bool in = i < have;
  long r = i;
  if (in) {
    if (rows)
      r = rows[off + i];
    else
      in = row_counts(a, r);
  }
  copy_row(dst + i * ldd, src + r * ld, (long)blockIdx.y * 1024, D, in, lane);
  if (again) copy_row(dst + (i + again) * ldd, src + r * ld, (long)blockIdx.y * 1024, D, in, lane);
}

// dst = src, rows of D values: a gradient that TMA could not write where the caller wants it.
__global__ void __launch_bounds__(256)
    vocab_copy_kernel(const __nv_bfloat16* __restrict__ src, long ld, long n, long D, __nv_bfloat16* __restrict__ dst,
                      long ldd) {
  grid_wait();
  grid_next();
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= n) return;
  copy_row(dst + i * ldd, src + i * ld, (long)blockIdx.y * 1024, D, true, threadIdx.x & 31);
}

// The row's (max, sum) in log2 units from its segments'; a fixed order over the threads t of `threads`. The two are kept
// apart: beside a large maximum (a finite mask on every token) f32 has no room for the logarithm of the sum, and the
// loss and the gradient need only differences to the maximum.
__device__ __forceinline__ float2 seg_fold(const float2* __restrict__ sr, long segs, int t, int threads) {
  float m = -INFINITY, s = 0.f;
  for (long q = t; q < segs; q += threads) {
    const float2 f = sr[q];
    const float hi = fmaxf(m, f.x);
    const float ref = hi == -INFINITY ? 0.f : hi;  // empty segments add their 0 (or NaN)
    s = s * exp2f(m - ref) + f.y * (f.x == -INFINITY ? 1.f : exp2f(f.x - ref));
    m = hi;
  }
  return make_float2(m, s);
}
__device__ __forceinline__ float2 seg_join(float2 a, float2 b) {
  const float hi = fmaxf(a.x, b.x), ref = hi == -INFINITY ? 0.f : hi;
  return make_float2(hi, a.y * (a.x == -INFINITY ? 1.f : exp2f(a.x - ref)) + b.y * (b.x == -INFINITY ? 1.f : exp2f(b.x - ref)));
}
__device__ __forceinline__ float2 warp_join(float2 v) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v = seg_join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
  return v;
}
__device__ __forceinline__ float2 seg_row(float2 v) { return make_float2(v.x == -INFINITY ? 0.f : v.x, v.y); }

// What the gradient needs of a row of the piece: info[i] = (max in log2 units, scale / T / sum; 0 where it does not
// count), and per answer entry the column (-1: absent) and the gradient there, in f32.
struct RowOut {
  float2* info;
  int* col;
  float* val;
};

// The logits of a row's answer entries, in log2 units: products of length D with gathered rows of W, summed in f32
// (the f16 terms would not do for the loss). Four entries to a warp, so that each value of x read serves four, and
// 16 to a block: rows with long lists are spread over blocks. Bound by the gathered rows, 2 D bytes an entry.
__global__ void __launch_bounds__(128)
    vocab_dots_kernel(const __nv_bfloat16* __restrict__ x, long ldx, const __nv_bfloat16* __restrict__ w, long ldw,
                      const __nv_bfloat16* __restrict__ bias, long V, long D, int K, const int* __restrict__ ids2,
                      float scale2, const int* __restrict__ rows, const int* __restrict__ count, long off,
                      float* __restrict__ uk) {
  grid_wait();
  grid_next();
  const long i = blockIdx.x;
  if (count && off + i >= *count) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long r = rows ? rows[off + i] : off + i;
  const int k0 = (blockIdx.y * 4 + warp) * 4;
  if (k0 >= K) return;
  const __nv_bfloat16* xr = x + i * ldx;
  const __nv_bfloat16* wr[4];
  int id[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    id[j] = k0 + j < K ? ids2[r * K + k0 + j] : -1;
    wr[j] = w + (id[j] >= 0 && id[j] < V ? (long)id[j] : 0L) * ldw;  // absent entries read row 0, to no effect
  }
  if ((id[0] & id[1] & id[2] & id[3]) < 0) return;
  const bool vec = ((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && ldx % 8 == 0 && ldw % 8 == 0;
  const long Dv = vec ? D / 8 * 8 : 0;
  float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (long c = lane * 8; c < Dv; c += 256) {
    const uint4 xv = *reinterpret_cast<const uint4*>(xr + c);
    uint4 wv[4];
#pragma unroll
    for (int j = 0; j < 4; j++) wv[j] = __ldg(reinterpret_cast<const uint4*>(wr[j] + c));
    const __nv_bfloat162* xh = reinterpret_cast<const __nv_bfloat162*>(&xv);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const float2 f = __bfloat1622float2(xh[q]);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 g = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&wv[j])[q]);
        d[j] = __fmaf_rn(f.x, g.x, d[j]);
        d[j] = __fmaf_rn(f.y, g.y, d[j]);
      }
    }
  }
  for (long c = Dv + lane; c < D; c += 32) {
    const float f = __bfloat162float(xr[c]);
#pragma unroll
    for (int j = 0; j < 4; j++) d[j] = __fmaf_rn(f, __bfloat162float(wr[j][c]), d[j]);
  }
  // the four sums in one butterfly: lane l ends with that of entry l / 8
  const bool hi = lane & 16, hi2 = lane & 8;
  const float a0 = (hi ? d[2] : d[0]) + __shfl_xor_sync(0xffffffffu, hi ? d[0] : d[2], 16);
  const float a1 = (hi ? d[3] : d[1]) + __shfl_xor_sync(0xffffffffu, hi ? d[1] : d[3], 16);
  float t = (hi2 ? a1 : a0) + __shfl_xor_sync(0xffffffffu, hi2 ? a0 : a1, 8);
#pragma unroll
  for (int o = 4; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int k = k0 + (lane >> 3);
  if ((lane & 7) == 0 && k < K) {
    const int c = ids2[r * K + k];
    uk[i * K + k] = __fmaf_rn(t, scale2, bias && c >= 0 && c < V ? vocab_bias2(__bfloat162float(bias[c]), scale2) : 0.f);
  }
}

// The sum of a row, or NaN while the device's error word holds a wait that ran out: its segments may not have been
// written, and nothing else tells the caller.
__device__ __forceinline__ float sum_or_nan(float s, const unsigned* err) { return err && *err ? NAN : s; }

// One warp per row: its lse from the segments, the loss, and what the gradient needs.
__device__ __forceinline__ void row_without(long r, long i, int K, int lane, float* loss, float* lse, const RowOut& o) {
  if (lane == 0) {
    loss[r] = 0.f;
    lse[r] = 0.f;
    if (o.info) o.info[i] = make_float2(0.f, 0.f);
  }
  if (o.info)
    for (int k = lane; k < K; k += 32) {
      o.col[i * K + k] = -1;
      o.val[i * K + k] = 0.f;
    }
}
// Cross entropy: the target's logit comes from the product itself (ut), so that loss = lse - u carries no difference
// between two ways of summing.
__global__ void __launch_bounds__(256)
    vocab_ce_rows_kernel(const int* __restrict__ target, long V, const float* __restrict__ row_scale,
                         const int* __restrict__ rows, const int* __restrict__ count, long off, long n,
                         const float2* __restrict__ stat, long ld_stat, const float* __restrict__ ut,
                         const unsigned* __restrict__ err, float* __restrict__ loss, float* __restrict__ lse,
                         RowOut o) {
  grid_wait();
  grid_next();
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= rows_here(count, off, n)) return;
  const long r = rows ? rows[off + i] : off + i;
  const int t = target[r];
  if (t < 0) return row_without(r, i, 1, lane, loss, lse, o);
  float2 ms = seg_row(warp_join(seg_fold(stat + i * ld_stat, ld_stat, lane, 32)));
  if (lane) return;
  ms.y = sum_or_nan(ms.y, err);
  float u = 0.f;
  if (t >= V)
    ms.y = NAN;  // a target past the vocabulary: seen in the loss
  else
    u = ut[i];
  const float log_sum = log2f(ms.y);
  loss[r] = ((ms.x - u) + log_sum) * kLn2;
  lse[r] = (ms.x + log_sum) * kLn2;
  if (o.info) {
    const float scale = row_scale ? row_scale[r] : 1.f;
    o.info[i] = make_float2(ms.x, scale == 0.f ? 0.f : scale / ms.y);
    o.col[i] = t;
    o.val[i] = (exp2f(u - ms.x) / ms.y - 1.f) * scale;
  }
}
// Distillation: ids2, p, ent of the teacher kernel, uk of the dots kernel. The p of a row sum to one, so the row's
// maximum is taken from every u before they are weighted.
__global__ void __launch_bounds__(256)
    vocab_distill_rows_kernel(long V, int K, const int* __restrict__ ids2, const float* __restrict__ p,
                              const float* __restrict__ ent, const uint8_t* __restrict__ has, float inv_t,
                              const float* __restrict__ row_scale, const int* __restrict__ rows,
                              const int* __restrict__ count, long off, long n, const float2* __restrict__ stat,
                              long ld_stat, const float* __restrict__ uk, const unsigned* __restrict__ err,
                              float* __restrict__ loss, float* __restrict__ lse, RowOut o) {
  grid_wait();
  grid_next();
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= rows_here(count, off, n)) return;
  const long r = rows ? rows[off + i] : off + i;
  if (!has[r]) return row_without(r, i, K, lane, loss, lse, o);
  float2 ms = seg_row(warp_join(seg_fold(stat + i * ld_stat, ld_stat, lane, 32)));
  ms.y = sum_or_nan(ms.y, err);
  const float scale = (row_scale ? row_scale[r] : 1.f) * inv_t;
  float acc = 0.f;
  bool bad = false;
  for (int k = lane; k < K; k += 32) {
    const int c = ids2[r * K + k];
    float val = 0.f;
    if (c >= V) {
      bad = true;
    } else if (c >= 0) {
      const float q = p[r * K + k], u = uk[i * K + k] - ms.x;
      if (!(q == 0.f)) acc = __fmaf_rn(-q, u, acc);
      val = (exp2f(u) / ms.y - q) * scale;
    }
    if (o.info) {
      o.col[i * K + k] = c;
      o.val[i * K + k] = val;
    }
  }
  acc = warp_sum_f(acc);
  if (__any_sync(0xffffffffu, bad)) ms.y = NAN;  // an id past the vocabulary: seen in the loss
  if (lane == 0) {
    const float log_sum = log2f(ms.y);
    loss[r] = (ent[r] + acc + log_sum) * kLn2;
    lse[r] = (ms.x + log_sum) * kLn2;
    if (o.info) o.info[i] = make_float2(ms.x, scale == 0.f ? 0.f : scale / ms.y);
  }
}

// Rows up to which the row tile has room for dz twice over: its bf16 values and, 64 rows below, the bf16 values of what
// their rounding took away (x is repeated there too). The products then carry 16 bits of dz for the price of 8: the
// row tile and, up to 32 rows, the k-block are no larger. With many rows single roundings average out; with few they
// stood out (12 rows: dx and dw off by 2.6e-3, bf16's own rounding of them 1.7e-3).
constexpr long kVocabLo = 64;

// The f16 terms of a tile of `rpb` rows x 256 NS columns become dz in place (bf16): t 2^(segment's max - max - 15)
// scale / sum, and at the answer's columns the f32 values of the rows kernels. A warp walks the rows, a lane owns 8
// columns of every 256. The block first lists the answer entries that fall into its tile (in an order that depends on
// nothing but the entries) and marks them in a bit mask; the walk leaves marked columns out, and the listed values are
// written after
// it. With `part` the column sums of the unrounded values go to part[row tile][V] for dbias. Rows from the count to
// the next multiple of 64 are zeroed (the weight-gradient product reads whole k-blocks of rows). With LO the rounding
// errors go, in bf16 too, to the rows kVocabLo below.
// Bound by HBM: 4 bytes per term.
constexpr int kDzScan = 16;  // answer entries of a block: 256 kDzScan at most
template <int NS>
struct DzSmem {
  static constexpr int COLS = 256 * NS;
  static size_t bytes(int rpb, long K, bool part) {
    return (size_t)rpb * COLS / 8 + (size_t)rpb * K * 8 + (part ? (size_t)8 * COLS * 4 : 0);
  }
  static size_t most(bool part) { return bytes(64, 256 * kDzScan / 64, part); }  // of every plan
};
template <int NS, bool PART, bool LO>
__global__ void __launch_bounds__(256, PART ? 3 : 4)
    vocab_dz_kernel(void* __restrict__ terms, long ld, long V, int K, const int* __restrict__ count, long off, long n,
                    int rpb, RowOut in, const float2* __restrict__ stat, long ld_stat, int seg_shift,
                    float* __restrict__ part) {
  constexpr long lo = LO ? kVocabLo : 0;
  grid_wait();
  grid_next();
  constexpr int COLS = 256 * NS;
  extern __shared__ __align__(16) uint8_t dyn_smem[];
  uint32_t* mask = reinterpret_cast<uint32_t*>(dyn_smem);                   // [rpb][COLS / 32]
  uint32_t* hit_at = mask + rpb * (COLS / 32);                              // [rpb K]: row << 16 | column
  float* hit_v = reinterpret_cast<float*>(hit_at + (long)rpb * K);          // [rpb K]
  float* fold = hit_v + (long)rpb * K;                                      // [8][COLS] (PART)
  __shared__ int warp_n[8];
  const long have = rows_here(count, off, n);
  const long r0 = (long)blockIdx.y * rpb, c0 = (long)blockIdx.x * COLS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* base = reinterpret_cast<uint16_t*>(terms) + r0 * ld + c0 + lane * 8;
  const int left = (int)min((long)COLS, V - c0) - lane * 8;  // columns from this lane's first on
  float sum[NS][8];
#pragma unroll
  for (int s = 0; s < NS; s++)
#pragma unroll
    for (int j = 0; j < 8; j++) sum[s][j] = 0.f;
  int hits = 0;
  const int nr = (int)max(0L, min((long)rpb, have - r0));
  if (nr > 0) {
    for (int q = threadIdx.x; q < rpb * (COLS / 32); q += 256) mask[q] = 0u;
    const int total = nr * K;
    const int* cols = in.col + r0 * K;
    const int width = (int)min((long)COLS, V - c0);
    uint32_t found = 0;  // bit 4 i + j: entry 4 (threadIdx.x + 256 i) + j lies in the tile
    int4 e[kDzScan / 4];
#pragma unroll
    for (int i = 0; i < kDzScan / 4; i++) {
      const int q = 4 * (threadIdx.x + 256 * i);
      if (q < total) e[i] = __ldg(reinterpret_cast<const int4*>(cols + q));  // the list's rows go on past `total`
    }
#pragma unroll
    for (int i = 0; i < kDzScan / 4; i++) {
      const int q = 4 * (threadIdx.x + 256 * i);
      if (q < total && (unsigned)(e[i].x - (int)c0) < (unsigned)width) found |= 1u << (4 * i);
      if (q + 1 < total && (unsigned)(e[i].y - (int)c0) < (unsigned)width) found |= 2u << (4 * i);
      if (q + 2 < total && (unsigned)(e[i].z - (int)c0) < (unsigned)width) found |= 4u << (4 * i);
      if (q + 3 < total && (unsigned)(e[i].w - (int)c0) < (unsigned)width) found |= 8u << (4 * i);
    }
    const int mine = __popc(found);
    // exclusive prefix over the threads
    int pre = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += t;
    }
    if (lane == 31) warp_n[warp] = pre;
    __syncthreads();
    int at = pre - mine;
#pragma unroll
    for (int q = 0; q < 8; q++) {
      if (q < warp) at += warp_n[q];
      hits += warp_n[q];
    }
    for (; found; found &= found - 1) {
      const int i = __ffs(found) - 1;
      hit_at[at++] = 4 * (threadIdx.x + 256 * (i >> 2)) + (i & 3);
    }
    __syncthreads();
    for (int h = threadIdx.x; h < hits; h += 256) {
      const uint32_t q = hit_at[h], row = q / (uint32_t)K, d = __ldg(cols + q) - (int)c0;
      hit_at[h] = row << 16 | d;
      hit_v[h] = in.val[r0 * K + q];
      atomicOr(&mask[row * (COLS / 32) + (d >> 5)], 1u << (d & 31));
    }
    __syncthreads();
#pragma unroll 2
    for (int q = warp; q < nr; q += 8) {
      const float2 f = __ldg(in.info + r0 + q);  // (max, scale / sum)
      uint4* at4 = reinterpret_cast<uint4*>(base + q * ld);
      const float2* sr = stat + (r0 + q) * ld_stat;
      uint4 raw[NS];
      float m[NS];
#pragma unroll
      for (int s = 0; s < NS; s++)
        if (256 * s < left) {  // V's pad up to a multiple of 8 lies inside ld
          raw[s] = at4[32 * s];
          m[s] = __ldg(&sr[(int)(c0 + 256 * s + lane * 8) >> seg_shift].x);
        }
#pragma unroll
      for (int s = 0; s < NS; s++) {
        if (256 * s >= left) continue;
        const uint32_t bits = mask[q * (COLS / 32) + 8 * s + (lane >> 2)] >> (8 * (lane & 3)) & 0xffu;
        if (__any_sync(__activemask(), bits)) {  // rare: columns whose values are listed
          uint32_t* t = reinterpret_cast<uint32_t*>(&raw[s]);
#pragma unroll
          for (int j = 0; j < 4; j++) t[j] &= ~((bits >> (2 * j) & 1u) * 0xffffu | (bits >> (2 * j + 1) & 1u) * 0xffff0000u);
        }
        // a row that does not count has scale 0 (its x is zero, so its terms are finite)
        const float k = m[s] == -INFINITY || f.y == 0.f ? 0.f : ex2(m[s] - f.x - 15.f) * f.y;
        const float2 k2 = make_float2(k, k);
        const __half2* h = reinterpret_cast<const __half2*>(&raw[s]);
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __fmul2_rn(__half22float2(h[j]), k2);
        uint4 o;
        uint32_t* u = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const __nv_bfloat162 b = __float22bfloat162_rn(v[j]);
          u[j] = *reinterpret_cast<const uint32_t*>(&b);
          if (PART) {
            sum[s][2 * j] += v[j].x;
            sum[s][2 * j + 1] += v[j].y;
          }
        }
        at4[32 * s] = o;
        if constexpr (LO) {  // what the rounding took away, `lo` rows below
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 h = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[j]));
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[j].x - h.x, v[j].y - h.y);
            u[j] = *reinterpret_cast<const uint32_t*>(&b);
          }
          *reinterpret_cast<uint4*>(base + (q + lo) * ld + 256 * s) = o;
        }
      }
    }
  }
  for (long q = nr + warp; q < min((long)rpb, (have + 63) / 64 * 64 - r0); q += 8)
#pragma unroll
    for (int s = 0; s < NS; s++)
      if (256 * s < left) {
        reinterpret_cast<uint4*>(base + q * ld)[32 * s] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (LO) reinterpret_cast<uint4*>(base + (q + lo) * ld)[32 * s] = make_uint4(0u, 0u, 0u, 0u);
      }
  if (PART) {
#pragma unroll
    for (int s = 0; s < NS; s++)
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<float4*>(fold + warp * COLS + 256 * s + lane * 8 + j) =
            make_float4(sum[s][j], sum[s][j + 1], sum[s][j + 2], sum[s][j + 3]);
  }
  __syncthreads();
  uint16_t* tile = reinterpret_cast<uint16_t*>(terms) + r0 * ld + c0;
  for (int h = threadIdx.x; h < hits; h += 256) {
    uint16_t* at = tile + (hit_at[h] >> 16) * ld + (hit_at[h] & 0xffffu);
    const __nv_bfloat16 b = __float2bfloat16_rn(hit_v[h]);
    *at = __bfloat16_as_ushort(b);
    if constexpr (LO) at[lo * ld] = __bfloat16_as_ushort(__float2bfloat16_rn(hit_v[h] - __bfloat162float(b)));
  }
  if constexpr (PART) {
    // thread t owns the block's columns t, t + 256, ...
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int c = 256 * s + threadIdx.x;
      float t = fold[c];
#pragma unroll
      for (int q = 1; q < 8; q++) t += fold[q * COLS + c];
      fold[c] = t;
    }
    __syncthreads();
    // The first listed value of a column adds all of that column's. Quadratic in the values listed: nothing beside the
    // walk when a row's answers are spread over the vocabulary, but not when they crowd into one tile (4,096 x 65,537 x
    // 1,024 with a bias, the whole call: 64 answers a row spread evenly 1,675 us, by Zipf's law 2,003, all among the
    // first 1,024 tokens 2,547; 20 answers 1,434, 1,445 and 1,635).
    for (int h = threadIdx.x; h < hits; h += 256) {
      const uint32_t c = hit_at[h] & 0xffffu;
      float t = 0.f;
      bool first = true;
      for (int g = 0; g < hits; g++) {
        const bool same = (hit_at[g] & 0xffffu) == c;
        first = first && !(same && g < h);
        t += same ? hit_v[g] : 0.f;
      }
      if (first) fold[c] += t;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; s++) {
      const int c = 256 * s + threadIdx.x;
      if (c0 + c < V) part[(long)blockIdx.y * V + c0 + c] = fold[c];
    }
  }
}

// sum (+)= the row tiles' column sums; on the last piece dbias = sum (f32 or bf16). 32 columns to a block, S slices of
// the tiles, both folded in a fixed order.
template <int S>
__global__ void __launch_bounds__(32 * S)
    vocab_dbias_kernel(const float* __restrict__ part, int tiles, long V, float* __restrict__ acc, int first, int last,
                       int f32, void* __restrict__ dbias) {
  grid_wait();
  grid_next();
  __shared__ float scr[S][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long v = (long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (v < V) {
#pragma unroll 8
    for (int q = slice; q < tiles; q += S) s += part[(long)q * V + v];
  }
  scr[slice][lane] = s;
  __syncthreads();
  if (slice || v >= V) return;
#pragma unroll
  for (int q = 1; q < S; q++) s += scr[q][lane];
  if (!first) s += acc[v];
  if (!last)
    acc[v] = s;
  else if (f32)
    reinterpret_cast<float*>(dbias)[v] = s;
  else
    reinterpret_cast<__nv_bfloat16*>(dbias)[v] = __float2bfloat16_rn(s);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint4 o;
  uint32_t* u = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    u[j] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return o;
}

// A lane's eight values of a sliced product at row `row` (plus, with `lo`, that many rows below), columns [c, c + 8).
// SPLIT: the block's warps share the slices and warp 0 has the sums (added in a fixed order). False where the lane has
// nothing to write.
template <bool SPLIT>
__device__ __forceinline__ bool slices_of(const SliceShape& s, const float* out, long ldo, const float* slabs, int bm,
                                          int bn, long row, long lo, long c, long D, float (&v)[8]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if constexpr (!SPLIT) {
    if (c >= D) return false;
    slice_sum8(s, out, ldo, slabs, bm, bn, row, (int)c, v, 0, 1);
    if (lo) {
      float l[8];
      slice_sum8(s, out, ldo, slabs, bm, bn, row + lo, (int)c, l, 0, 1);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += l[j];
    }
    return true;
  } else {
    __shared__ float part[8][256];
    if (c < D) {
      slice_sum8(s, out, ldo, slabs, bm, bn, row, (int)c, v, warp, 8);
      if (lo) {
        float l[8];
        slice_sum8(s, out, ldo, slabs, bm, bn, row + lo, (int)c, l, warp, 8);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] += l[j];
      }
      *reinterpret_cast<float4*>(&part[warp][lane * 8]) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(&part[warp][lane * 8 + 4]) = make_float4(v[4], v[5], v[6], v[7]);
    }
    __syncthreads();
    if (warp || c >= D) return false;
#pragma unroll
    for (int q = 1; q < 8; q++)
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += part[q][lane * 8 + j];
    return true;
  }
}

// dx row rows[off + i] = row i of the sliced product dz W, in bf16. With one answer per row (K = 1) its column of dz
// carries most of the row, and what its rounding to bf16 took away (val - bf16(val)) W[target] is given back, so that
// dx is rounded once; among many answers no single rounding stands out. With `lo` the product's row lo + i holds what
// dz's rounding took from row i. One warp per row and 256
// columns, or (SPLIT, for many slices) one block, its warps taking every eighth slice.
template <bool SPLIT>
__global__ void __launch_bounds__(256)
    vocab_dx_kernel(const float* __restrict__ out, long ldo, const float* __restrict__ slabs, int bm, int bn, int grid,
                    const int* __restrict__ rows, const int* __restrict__ count, long off, long n, long V, long D,
                    long lo, int K, RowOut in, const __nv_bfloat16* __restrict__ w, long ldw,
                    __nv_bfloat16* __restrict__ dx, long lddx) {
  grid_wait();
  grid_next();
  const long i = SPLIT ? blockIdx.x : (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long have = rows_here(count, off, n);
  if (i >= have) return;
  const SliceShape shape = slice_shape((int)(lo ? 2 * lo : have), (int)D, (int)V, bm, bn, grid);
  const long r = rows ? rows[off + i] : off + i;
  const bool vec = ((uintptr_t)dx & 15) == 0 && lddx % 8 == 0 && D % 8 == 0;
  __nv_bfloat16* d = dx + r * lddx;
  float rest = 0.f;
  const __nv_bfloat16* wr = w;
  if (K == 1 && !lo && in.col[i] >= 0 && in.col[i] < V) {
    rest = in.val[i] - __bfloat162float(__float2bfloat16_rn(in.val[i]));
    wr = w + (long)in.col[i] * ldw;
  }
  const bool wvec = ((uintptr_t)w & 15) == 0 && ldw % 8 == 0;
  const long c = (long)blockIdx.y * 256 + lane * 8;
  float v[8];
  if (!slices_of<SPLIT>(shape, out, ldo, slabs, bm, bn, i, lo, c, D, v)) return;
  if (rest != 0.f) {
    if (wvec && c + 8 <= D) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(wr + c));
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 f = __bfloat1622float2(h[j]);
        v[2 * j] = __fmaf_rn(rest, f.x, v[2 * j]);
        v[2 * j + 1] = __fmaf_rn(rest, f.y, v[2 * j + 1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (c + j < D) v[j] = __fmaf_rn(rest, __bfloat162float(wr[c + j]), v[j]);
    }
  }
  if (vec) {
    *reinterpret_cast<uint4*>(d + c) = pack8(v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + j < D) d[c + j] = __float2bfloat16_rn(v[j]);
  }
}

// The weight gradient from f32: a sliced product's parts (slabs) or the sum of the pieces (slabs NULL, src = acc);
// pieces before the last are kept in acc, the last goes to dw in the caller's type. One warp per row and 256 columns,
// or one block (SPLIT).
template <bool SPLIT>
__global__ void __launch_bounds__(256)
    vocab_dw_kernel(const float* __restrict__ src, long lds, const float* __restrict__ slabs, int bm, int bn, int grid,
                    const int* __restrict__ count, long off, long n, float* __restrict__ acc, int add, int last, long V,
                    long D, int f32, void* __restrict__ dw, long lddw) {
  grid_wait();
  grid_next();
  const long r = SPLIT ? blockIdx.x : (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long c = (long)blockIdx.y * 256 + (threadIdx.x & 31) * 8;
  if (r >= V) return;
  float v[8];
  if (slabs) {
    const SliceShape shape = slice_shape((int)V, (int)D, (int)rows_here(count, off, n), bm, bn, grid);
    if (!slices_of<SPLIT>(shape, src, lds, slabs, bm, bn, r, 0, c, D, v)) return;
  } else {
    if (c >= D) return;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = src[r * lds + c + j];
  }
  if (add) {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += acc[r * lds + c + j];
  }
  if (!last) {
#pragma unroll
    for (int j = 0; j < 8; j++) acc[r * lds + c + j] = v[j];
  } else if (f32) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + j < D) reinterpret_cast<float*>(dw)[r * lddw + c + j] = v[j];
  } else {
    __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(dw) + r * lddw + c;
    if (((uintptr_t)dw & 15) == 0 && lddw % 8 == 0 && c + 8 <= D) {
      *reinterpret_cast<uint4*>(d) = pack8(v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (c + j < D) d[j] = __float2bfloat16_rn(v[j]);
    }
  }
}

// ---------------------------------------------------------------------------------------------- host side
// Rows up to which one row tile holds them all: leaving rows out of the products then saves nothing, so no plan is
// made (two launches fewer; the rows without an answer are zeroed instead).
constexpr long kVocabOneTile = 128;
// Weights whose rows do not start at 128-byte lines cost the products' TMA boxes an extra line each. For the three
// products of a gradient a copy with padded rows pays for itself with enough rows: V = 50,048, 4,096 rows,
// D = 520 / 1,000 / 2,056: 930 / 1,100 / 2,233 us with the copy, 1,114 / 1,108 / 2,328 without; 1,000 rows: 270 / 352 /
// 678 and 275 / 323 / 598. One number for every D is a compromise: on straight lines between these figures the two meet
// below 1,000 rows at D = 520, near 3,400 at D = 1,000 and near 2,400 at D = 2,056. For the loss alone the copy does not
// pay (4,096 rows: 282 / 341 / 761 and 274 / 310 / 676).
constexpr long kVocabPackRows = 2048;
// Rows up to which the weight gradient (V x D values out, a short inner axis) is bound by its writes and goes out from
// registers: V = 118,208, D = 3,712, 5 / 256 rows: the whole call 522 / 719 us, 556 / 737 through shared memory and
// TMA stores; from 1,024 rows on the two do not differ.
constexpr long kVocabDirectRows = 512;
// Bytes of terms that one piece may hold. Fewer pieces mean fewer passes over the f32 weight gradient (each piece
// after the first adds to it: 8 V D bytes). 4,096 x 65,537 x 1,024 in one piece / in two: 1.54-1.71 / 2.20-2.26 ms with
// a bf16 weight gradient, 1.62-1.76 / 1.93-2.07 ms with an f32 one.
constexpr size_t kVocabPieceBytes = (size_t)4 << 30;
constexpr int kSplitSlices = 8;     // slices of a product that one warp still adds up by itself
constexpr size_t kVocabMaxK = 512;  // entries of a row: its lists stay in shared memory

struct VocabPlan {
  bool compact, pack_x, pack_w;
  long lo;         // rows below dz where its rounding errors go (0: nowhere)
  bool dw_slice;   // dW by a sliced product
  bool dw_copy;    // dW in padded rows, then copied to the caller's
  long Dp;         // row stride of the packed matrices and of the f32 products
  long ldt;        // row stride of the terms
  int bn;          // column tile of the logits product
  int bd;          // column tile of the two products over D columns
  long ld_stat;
  long R;          // rows of a piece
  int pieces;
  int rpb;         // rows of a block that turns terms into gradients
  int ns;          // its columns, in 256s
  size_t bytes;
  // offsets into the workspace
  size_t ids2, p, ent, has, rows, count, xp, wp, stat, ut, uk, terms, info, col, val, dxs, slabs, dws, dwacc, part, dbacc;
};

static size_t carve(size_t& at, size_t bytes) {
  const size_t o = at;
  at += (bytes + 255) / 256 * 256;
  return o;
}

// K = 0: cross entropy. x_ok, w_ok: the matrix starts at 16 bytes and its row stride is a multiple of 8 (what TMA
// needs); w_lines: the same for 128 bytes and 64. dw_copy: the bf16 weight gradient cannot be written by TMA.
static VocabPlan vocab_plan(long N, long V, long D, long K, bool bias, bool grad, bool x_ok, bool w_ok, bool w_lines,
                            bool dw_copy, size_t piece_bytes, int sms) {
  VocabPlan p{};
  const long k1 = K ? K : 1;
  p.compact = N > kVocabOneTile;
  p.pack_x = p.compact || grad || !x_ok;
  p.lo = grad && N <= kVocabLo ? kVocabLo : 0;
  p.pack_w = !w_ok || (!w_lines && grad && N >= kVocabPackRows);
  p.Dp = round_up(D, 64);
  p.ldt = round_up(V, 64);
  p.bn = V > 148 * 128 ? 256 : 128;
  p.bd = D > 128 ? 256 : 128;
  p.ld_stat = ceil_div(V, p.bn) * 2;
  if (!piece_bytes) piece_bytes = kVocabPieceBytes;
  long R = (long)(piece_bytes / ((size_t)p.ldt * 2)) / 128 * 128;
  if (R < 128) R = 128;
  if (R > round_up(N, 128)) R = round_up(N, 128);
  if (R > (1 << 18)) R = 1 << 18;  // 8-row tiles on a grid's second axis
  p.pieces = (int)ceil_div(N, R);
  p.R = round_up(ceil_div(N, p.pieces), 128);
  p.pieces = (int)ceil_div(N, p.R);
  // a weight gradient of fewer 256 x 256 tiles than there are pairs of SMs, over enough rows to be cut
  p.dw_slice = ceil_div(V, 256) * ceil_div(D, 256) < sms / 2 && p.R >= 512;
  // 64 x 1,024 terms to a block, fewer where that leaves SMs idle, lists more than 512 answers or has no room for
  // all of its rows' entries (they may all name one tile)
  p.ns = ceil_div(V, 1024) * ceil_div(N, 64) >= 2 * sms ? 4 : 1;
  p.rpb = 64;
  const long cols = 256L * p.ns;
  while (p.rpb > 8 && (p.rpb * k1 > 256 * kDzScan || ceil_div(V, cols) * ceil_div(N, p.rpb) < 2 * sms ||
                       (double)p.rpb * k1 * (V < cols ? 1.0 : (double)cols / V) > 512.0))
    p.rpb /= 2;
  size_t at = 0;
  if (K) {
    p.ids2 = carve(at, (size_t)N * K * 4);
    p.p = carve(at, (size_t)N * K * 4);
    p.ent = carve(at, (size_t)N * 4);
    p.has = carve(at, (size_t)N);
  }
  if (p.compact) {
    p.rows = carve(at, (size_t)N * 4);
    p.count = carve(at, 4);
  }
  if (p.pack_x) p.xp = carve(at, (size_t)p.R * p.Dp * 2);
  if (p.pack_w) p.wp = carve(at, (size_t)round_up(V, 64) * p.Dp * 2);
  p.stat = carve(at, (size_t)p.R * p.ld_stat * 8);
  if (K)
    p.uk = carve(at, (size_t)p.R * K * 4);
  else
    p.ut = carve(at, (size_t)p.R * 4);
  if (grad) {
    p.terms = carve(at, (size_t)p.R * p.ldt * 2);
    p.info = carve(at, (size_t)p.R * 8);
    p.col = carve(at, (size_t)p.R * k1 * 4);
    p.val = carve(at, (size_t)p.R * k1 * 4);
    p.dxs = carve(at, (size_t)p.R * p.Dp * 4);
    p.slabs = carve(at, (size_t)kSliceSlabs * sms * 128 * p.bd * 4);
    p.dw_copy = dw_copy && !p.dw_slice && p.pieces == 1;
    if (p.dw_slice || p.dw_copy) p.dws = carve(at, (size_t)V * p.Dp * (p.dw_slice ? 4 : 2));
    if (p.pieces > 1) p.dwacc = carve(at, (size_t)V * p.Dp * 4);
    if (bias) {
      p.part = carve(at, (size_t)(p.R / p.rpb) * V * 4);
      p.dbacc = carve(at, (size_t)V * 4);
    }
  }
  p.bytes = at;
  return p;
}

struct VocabCall {
  const char* what;
  const void* x;
  size_t ldx;
  const void* w;
  size_t ldw;
  const void* bias;
  const int* ids;
  const float* teacher;
  size_t K;  // 0: cross entropy, ids holds one target per row
  double temperature;
  const float* row_scale;
  size_t N, V, D;
  float *loss, *lse;
  void* dx;
  size_t lddx;
  void* dw;
  size_t lddw;
  void* dbias;
  int dw_f32;
  size_t piece_bytes;
  void* ws;
  size_t ws_bytes;
  cudaStream_t st;
  bool grad;
};

static bool rows16(const void* p, size_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }
static bool rows128(const void* p, size_t ld) { return ((uintptr_t)p & 127) == 0 && ld % 64 == 0; }

template <int NS, bool PART, bool LO>
static int dz_launch(const VocabPlan& p, uint8_t* ws, long V, long K, const int* count, long off, long n, RowOut ro,
                     float* part, cudaStream_t st) {
  const size_t smem = DzSmem<NS>::bytes(p.rpb, K, PART);
  // once per device, to what the largest call needs: another thread's call may launch the same kernel at any time
  const int rc = raise_smem((const void*)vocab_dz_kernel<NS, PART, LO>, DzSmem<NS>::most(PART));
  if (rc) return rc;
  const dim3 grid((unsigned)ceil_div(V, 256 * NS), (unsigned)(round_up(n, 64) / p.rpb));
  PL_CUDA(launch_early(vocab_dz_kernel<NS, PART, LO>, grid, 256, smem, st, ws + p.terms, p.ldt, V, (int)K, count, off, n, p.rpb, ro,
                       (const float2*)(ws + p.stat), p.ld_stat, p.bn == 256 ? 7 : 6, part));
  count_launch();
  return PL_OK;
}

static int vocab_run(const VocabCall& c) {
  PL_REQUIRE(c.V > 0 && c.D > 0, PL_ERR_INVALID, "%s: V = %zu, D = %zu", c.what, c.V, c.D);
  PL_REQUIRE(c.N <= (1u << 30) && c.V <= (1u << 30) && c.D <= (1u << 22), PL_ERR_INVALID,
             "%s: N = %zu, V = %zu, D = %zu is too large", c.what, c.N, c.V, c.D);
  PL_REQUIRE(c.K <= kVocabMaxK, PL_ERR_INVALID, "%s: K = %zu entries, at most %zu", c.what, c.K, kVocabMaxK);
  PL_REQUIRE(c.ldx >= c.D && c.ldw >= c.D, PL_ERR_INVALID, "%s: row strides %zu, %zu below D = %zu", c.what, c.ldx, c.ldw,
             c.D);
  PL_REQUIRE(c.temperature > 0.0 && c.temperature < 1e30, PL_ERR_INVALID, "%s: temperature %g", c.what, c.temperature);
  PL_REQUIRE(c.w, PL_ERR_INVALID, "%s: NULL weights", c.what);
  if (c.grad) {
    PL_REQUIRE(c.dw, PL_ERR_INVALID, "%s: NULL weight gradient", c.what);
    PL_REQUIRE(c.lddx >= c.D && c.lddw >= c.D, PL_ERR_INVALID, "%s: gradient row strides %zu, %zu below D = %zu", c.what,
               c.lddx, c.lddw, c.D);
    PL_REQUIRE(!c.bias == !c.dbias, PL_ERR_INVALID, "%s: bias and its gradient go together", c.what);
  }
  PL_REQUIRE(c.N == 0 || (c.x && c.ids && (!c.K || c.teacher) && c.loss && c.lse && (!c.grad || c.dx)), PL_ERR_INVALID,
             "%s: NULL matrix or answers", c.what);
  int rc = require_device();
  if (rc) return rc;
  const long N = (long)c.N, V = (long)c.V, D = (long)c.D, K = (long)c.K, k1 = K ? K : 1;
  cudaStream_t st = c.st;
  const size_t wsize = c.dw_f32 ? 4 : 2;
  if (N == 0) {
    if (c.grad) {
      PL_CUDA(cudaMemset2DAsync(c.dw, c.lddw * wsize, 0, c.D * wsize, c.V, st));
      if (c.dbias) PL_CUDA(cudaMemsetAsync(c.dbias, 0, c.V * wsize, st));
    }
    return PL_OK;
  }
  const int sms = gemm_sms();
  const VocabPlan p = vocab_plan(N, V, D, K, c.bias != nullptr, c.grad, rows16(c.x, c.ldx), rows16(c.w, c.ldw),
                                 rows128(c.w, c.ldw), c.grad && !c.dw_f32 && !rows16(c.dw, c.lddw),
                                 c.piece_bytes, sms);
  PL_REQUIRE(c.ws && c.ws_bytes >= p.bytes && ((uintptr_t)c.ws & 255) == 0, PL_ERR_INVALID,
             "%s: %zu bytes of workspace (256-byte aligned), %zu needed", c.what, c.ws ? c.ws_bytes : (size_t)0, p.bytes);
  uint8_t* ws = (uint8_t*)c.ws;
  int* rows = p.compact ? (int*)(ws + p.rows) : nullptr;
  int* count = p.compact ? (int*)(ws + p.count) : nullptr;
  const float inv_t = (float)(1.0 / c.temperature);
  const float scale2 = (float)((double)kLog2e / c.temperature);
  const __nv_bfloat16* bias = (const __nv_bfloat16*)c.bias;
  const unsigned* err = device_error_word();
  Answers a{K ? nullptr : c.ids, K ? ws + p.has : nullptr};
  if (K) {
    const size_t smem = (size_t)4 * 2 * round_up(K, 4) * 4;
    PL_CUDA(launch_early(vocab_teacher_kernel, (unsigned)ceil_div(N, 4), 128, smem, st, c.ids, c.teacher, N, (int)K,
                         scale2, (int*)(ws + p.ids2), (float*)(ws + p.p), (float*)(ws + p.ent), ws + p.has));
    count_launch();
  }
  if (p.compact) {
    if (c.grad) PL_CUDA(cudaMemset2DAsync(c.dx, c.lddx * 2, 0, c.D * 2, c.N, st));  // rows that do not count
    PL_CUDA(launch_early(vocab_plan_kernel, 1, 1024, 0, st, a, N, rows, count, c.loss, c.lse));
    count_launch();
  }
  const __nv_bfloat16* w = (const __nv_bfloat16*)c.w;
  long ldw = (long)c.ldw;
  if (p.pack_w) {
    __nv_bfloat16* wp = (__nv_bfloat16*)(ws + p.wp);
    PL_CUDA(launch_early(vocab_pack_kernel, dim3((unsigned)ceil_div(round_up(V, 64), 8), (unsigned)ceil_div(D, 1024)),
                         256, 0, st, w, ldw, D, Answers{}, nullptr, nullptr, 0, V, wp, p.Dp, 0));
    count_launch();
    w = wp;
    ldw = p.Dp;
  }
  const long lo = p.lo;  // (then one piece, no plan)
  for (int q = 0; q < p.pieces; q++) {
    const long off = (long)q * p.R, n = N - off < p.R ? N - off : p.R;
    const long n2 = lo ? 2 * lo : n;  // rows of the products with dz
    const __nv_bfloat16* x = (const __nv_bfloat16*)c.x;  // without a plan there is one piece
    long ldx = (long)c.ldx;
    if (p.pack_x) {
      __nv_bfloat16* xp = (__nv_bfloat16*)(ws + p.xp);
      const dim3 grid((unsigned)ceil_div(round_up(n, 64), 8), (unsigned)ceil_div(D, 1024));
      PL_CUDA(launch_early(vocab_pack_kernel, grid, 256, 0, st, x, ldx, D, a, rows, count, off, n, xp, p.Dp, lo));
      count_launch();
      x = xp;
      ldx = p.Dp;
    }
    // logits: statistics of every segment, the targets' logits, and the terms
    const Operand X{x, p.pack_x ? p.R : n, D, ldx, 1, 0}, W{w, V, D, ldw, 1, 0};
    {
      EpiArgs e{};
      e.pdl = 1;
      e.out = c.grad ? ws + p.terms : nullptr;
      e.ldo = p.ldt;
      e.out_rows = (int)n;
      e.out_cols = (int)V;
      // The tensor core's accumulator truncates: over steps of 16 products a logit loses on average D 2^-30 of itself
      // (measured over D = 64 .. 8,192, hidden states that lean towards the weight row or not: 0.9 .. 1.0e-9 D), which
      // at D = 4,096 is 4e-6, many times what rounding to nearest would leave. The scale gives that back; what remains
      // is 2e-7 .. 7e-7.
      e.scale2 = (float)((double)kLog2e / c.temperature * (1.0 + (double)D / (1 << 30)));
      e.bias_scale2 = scale2;
      e.vbias = bias;
      e.stat = (float2*)(ws + p.stat);
      e.ld_stat = p.ld_stat;
      if (!K) {
        e.target = c.ids;
        e.row_ids = rows ? rows + off : nullptr;
        e.ut = (float*)(ws + p.ut);
      }
      e.dyn_rows = count;
      e.dyn_off = (int)off;
      rc = gemm_launch(p.bn, EPI_VOCAB, false, false, X, W, (int)n, (int)V, (int)D, 1, e, st);
      if (rc) return rc;
    }
    RowOut ro{};
    if (c.grad) ro = RowOut{(float2*)(ws + p.info), (int*)(ws + p.col), (float*)(ws + p.val)};
    if (K) {
      PL_CUDA(launch_early(vocab_dots_kernel, dim3((unsigned)n, (unsigned)ceil_div(K, 16)), 128, 0, st, x, ldx, w,
                           ldw, bias, V, D, (int)K, (const int*)(ws + p.ids2), scale2, rows, count, off,
                           (float*)(ws + p.uk)));
      count_launch();
      PL_CUDA(launch_early(vocab_distill_rows_kernel, (unsigned)ceil_div(n, 8), 256, 0, st, V, (int)K,
                           (const int*)(ws + p.ids2), (const float*)(ws + p.p), (const float*)(ws + p.ent),
                           ws + p.has, inv_t, c.row_scale, rows, count, off, n, (const float2*)(ws + p.stat),
                           p.ld_stat, (const float*)(ws + p.uk), err, c.loss, c.lse, ro));
    } else {
      PL_CUDA(launch_early(vocab_ce_rows_kernel, (unsigned)ceil_div(n, 8), 256, 0, st, c.ids, V, c.row_scale, rows,
                           count, off, n, (const float2*)(ws + p.stat), p.ld_stat, (const float*)(ws + p.ut), err,
                           c.loss, c.lse, ro));
    }
    count_launch();
    if (!c.grad) continue;
    const bool last = q == p.pieces - 1;
    float* part = bias ? (float*)(ws + p.part) : nullptr;
    const auto wide = lo ? (bias ? dz_launch<4, true, true> : dz_launch<4, false, true>)
                         : (bias ? dz_launch<4, true, false> : dz_launch<4, false, false>);
    const auto narrow = lo ? (bias ? dz_launch<1, true, true> : dz_launch<1, false, true>)
                           : (bias ? dz_launch<1, true, false> : dz_launch<1, false, false>);
    const auto dz = p.ns == 4 ? wide : narrow;
    rc = dz(p, ws, V, k1, count, off, n, ro, part, st);
    if (rc) return rc;
    if (bias) {
      const int tiles = (int)(round_up(n, 64) / p.rpb);
      // a few dozen tiles: eight loads to a thread; thousands (many rows of a small vocabulary): more threads
      const bool few = tiles <= 256;
      PL_CUDA(launch_early(few ? vocab_dbias_kernel<8> : vocab_dbias_kernel<32>, (unsigned)ceil_div(V, 32),
                           few ? 256 : 1024, 0, st, part, tiles, V, (float*)(ws + p.dbacc), q == 0, last, c.dw_f32,
                           c.dbias));
      count_launch();
    }
    float* slabs = (float*)(ws + p.slabs);
    {  // dx = dz W
      EpiArgs g{};
      g.pdl = 1;
      g.out = ws + p.dxs;
      g.ldo = p.Dp;
      g.slabs = slabs;
      g.out_rows = (int)n2;
      g.out_cols = (int)D;
      g.dyn_rows = count;
      g.dyn_off = (int)off;
      const Operand Z{ws + p.terms, p.R, V, p.ldt, 1, 0};
      rc = gemm_launch(p.bd, EPI_SLICE, false, true, Z, W, (int)n2, (int)D, (int)V, 1, g, st);
      if (rc) return rc;
      const bool pairs = gemm_paired(p.bd, EPI_SLICE, false, true, (int)n2);
      const int bm = pairs ? 256 : 128, grid = pairs ? sms / 2 : sms;
      const bool split = slice_shape((int)n2, (int)D, (int)V, bm, p.bd, grid).q > kSplitSlices;
      PL_CUDA(launch_early((split ? vocab_dx_kernel<true> : vocab_dx_kernel<false>),
                           dim3((unsigned)(split ? n : ceil_div(n, 8)), (unsigned)ceil_div(D, 256)), 256, 0, st,
                           (const float*)(ws + p.dxs), p.Dp, slabs, bm, p.bd, grid, rows, count, off, n, V, D, lo,
                           (int)k1, ro, w, ldw, (__nv_bfloat16*)c.dx, (long)c.lddx));
      count_launch();
    }
    {  // dW (+)= dz^T x: to the caller's matrix, to the f32 sum of the pieces, or sliced
      EpiArgs g{};
      g.pdl = 1;
      g.alpha = 1.f;
      g.out_rows = (int)V;
      g.out_cols = (int)D;
      g.dyn_rows = count;
      g.dyn_off = (int)off;
      g.dyn_k = 1;
      const bool direct = !p.dw_slice && (p.pieces == 1 || c.dw_f32);
      const bool via = direct && p.dw_copy;  // in bf16 rows that TMA can write, then copied
      float* acc = (float*)(ws + p.dwacc);
      const bool rows32 = via || (((uintptr_t)c.dw & 31) == 0 && c.lddw % 16 == 0);
      const int bf16_out = rows32 && n <= kVocabDirectRows ? EPI_DIRECT : EPI_BF16;
      const int epi = p.dw_slice ? EPI_SLICE : (direct && !c.dw_f32 ? bf16_out : EPI_F32);
      g.out = p.dw_slice || via ? (void*)(ws + p.dws) : (direct ? c.dw : (void*)acc);
      g.ldo = direct && !via ? (long)c.lddw : p.Dp;
      g.slabs = slabs;
      g.accum = !p.dw_slice && q > 0;
      const Operand Xk{x, n2, D, ldx, 1, 0};
      const Operand Zk{ws + p.terms, n2, V, p.ldt, 1, 0};
      rc = gemm_launch(p.bd, epi, true, true, Zk, Xk, (int)V, (int)D, (int)n2, 1, g, st);
      if (rc) return rc;
      if (via) {
        PL_CUDA(launch_early(vocab_copy_kernel, dim3((unsigned)ceil_div(V, 8), (unsigned)ceil_div(D, 1024)), 256, 0,
                             st, (const __nv_bfloat16*)(ws + p.dws), p.Dp, V, D, (__nv_bfloat16*)c.dw,
                             (long)c.lddw));
        count_launch();
      }
      if (!direct && (p.dw_slice || last)) {
        const bool pairs = gemm_paired(p.bd, EPI_SLICE, true, true, (int)V);
        const int bm = pairs ? 256 : 128, grid = pairs ? sms / 2 : sms;
        const bool split = p.dw_slice && slice_shape((int)V, (int)D, (int)n, bm, p.bd, grid).q > kSplitSlices;
        PL_CUDA(launch_early((split ? vocab_dw_kernel<true> : vocab_dw_kernel<false>),
                             dim3((unsigned)(split ? V : ceil_div(V, 8)), (unsigned)ceil_div(D, 256)), 256, 0, st,
                              p.dw_slice ? (const float*)(ws + p.dws) : acc, p.Dp, p.dw_slice ? slabs : nullptr, bm,
                             p.bd, grid, count, off, n, acc, p.dw_slice && q > 0, last, V, D, c.dw_f32, c.dw,
                             (long)c.lddw));
        count_launch();
      }
    }
  }
  return PL_OK;
}

}  // namespace pl

extern "C" {

int pl_test_vocab_dz_smem(int* bytes) {
  cudaFuncAttributes a;
  PL_CUDA(cudaFuncGetAttributes(&a, (const void*)pl::vocab_dz_kernel<4, true, false>));
  *bytes = a.maxDynamicSharedSizeBytes;
  return PL_OK;
}

size_t pl_vocab_ws(size_t N, size_t V, size_t D, size_t K, uint8_t bias, uint8_t grad, uint8_t aligned,
                   size_t piece_bytes) {
  if (N == 0 || V == 0 || D == 0) return 0;
  const bool ok = aligned != 0;
  return pl::vocab_plan((long)N, (long)V, (long)D, (long)K, bias != 0, grad != 0, ok, ok, ok, !ok, piece_bytes,
                        pl::gemm_sms())
      .bytes;
}

int pl_vocab_ce_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* target,
                    size_t N, size_t V, size_t D, float* loss, float* lse, void* ws, size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_ce_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.ids = target;
  c.temperature = 1.0;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.st = (cudaStream_t)stream;
  return pl::vocab_run(c);
}

int pl_vocab_ce_grad_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* target,
                         const float* row_scale, size_t N, size_t V, size_t D, float* loss, float* lse, void* dx,
                         size_t lddx, void* dw, size_t lddw, void* dbias, uint8_t dw_f32, size_t piece_bytes, void* ws,
                         size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_ce_grad_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.ids = target;
  c.temperature = 1.0;
  c.row_scale = row_scale;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.dx = dx, c.lddx = lddx, c.dw = dw, c.lddw = lddw, c.dbias = dbias, c.dw_f32 = dw_f32, c.piece_bytes = piece_bytes;
  c.grad = true;
  c.st = (cudaStream_t)stream;
  return pl::vocab_run(c);
}

int pl_vocab_distill_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* ids,
                         const float* teacher, size_t K, double temperature, size_t N, size_t V, size_t D, float* loss,
                         float* lse, void* ws, size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_distill_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.ids = ids, c.teacher = teacher, c.K = K;
  c.temperature = temperature;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.st = (cudaStream_t)stream;
  if (K == 0) return pl::set_error(PL_ERR_INVALID, "pl_vocab_distill_dev: K = 0");
  return pl::vocab_run(c);
}

int pl_vocab_distill_grad_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* ids,
                              const float* teacher, size_t K, double temperature, const float* row_scale, size_t N,
                              size_t V, size_t D, float* loss, float* lse, void* dx, size_t lddx, void* dw, size_t lddw,
                              void* dbias, uint8_t dw_f32, size_t piece_bytes, void* ws, size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_distill_grad_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.ids = ids, c.teacher = teacher, c.K = K;
  c.temperature = temperature;
  c.row_scale = row_scale;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.dx = dx, c.lddx = lddx, c.dw = dw, c.lddw = lddw, c.dbias = dbias, c.dw_f32 = dw_f32, c.piece_bytes = piece_bytes;
  c.grad = true;
  c.st = (cudaStream_t)stream;
  if (K == 0) return pl::set_error(PL_ERR_INVALID, "pl_vocab_distill_grad_dev: K = 0");
  return pl::vocab_run(c);
}

}  // extern "C"
