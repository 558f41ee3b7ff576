// A large-vocabulary head and what it is trained with: softmax cross entropy against one target per row, and
// distillation from a teacher's top logits, forward and with gradients, without the logits ever being kept.
//
//   u = (x W^T + bias) / T          rows n < N, vocabulary v < V, hidden width D
//   lse_n = log sum_v exp u_nv      p_nk: the answer's probabilities (one entry of 1, or softmax(teacher / T))
//   loss_n = sum_k p_nk (log p_nk - u_n,id(n,k)) + lse_n
//   dz = scale_n / T (exp(u - lse) - sum_k p_nk onehot(id(n,k))),   dx = dz W,  dW = dz^T x,  dbias = sum_n dz
//
// Rows without an answer (a negative target, no entry present) are taken out before the products: a plan kernel
// lists the rows that count, the products' row extent is read from the device. One product gives the logits: its
// epilogue (pl_gemm.cuh, EPI_VOCAB) folds each row's 128 columns to (max, sum) and, when gradients are wanted,
// leaves 2^(u - max) in f16 in a buffer of as many rows as the workspace allows. Once the row's statistics are
// known these terms become dz in place (bf16, the one rounding of the gradient), and two more products give dx
// and dW. Three products of 2 N V D flops is also the least that the gradients need; recomputing the logits
// instead of keeping the terms would make it four.
#include <cuda_fp16.h>

#include "pl_common.cuh"
#include "pl_gemm.cuh"
#include "pl_runtime.h"

namespace pl {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The answers of a call: one target per row (ids [N], teacher NULL, K = 1) or K entries per row.
struct Answers {
  const int* ids;
  const float* teacher;  // NULL: every present entry has probability 1
  long K;
};

__device__ __forceinline__ bool row_counts(const Answers& a, long row) {
  for (long k = 0; k < a.K; k++) {
    if (a.ids[row * a.K + k] < 0) continue;
    if (!a.teacher || a.teacher[row * a.K + k] > -INFINITY || isnan(a.teacher[row * a.K + k])) return true;
  }
  return false;
}

// rows[0 .. *count) = the rows that count, in order; loss = lse = 0 for the others. One block.
__global__ void __launch_bounds__(1024)
    vocab_plan_kernel(Answers a, long N, int* __restrict__ rows, int* __restrict__ count, float* __restrict__ loss,
                      float* __restrict__ lse) {
  __shared__ int warp_n[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (long r0 = 0; r0 < N; r0 += 1024) {
    const long r = r0 + threadIdx.x;
    const bool in = r < N && row_counts(a, r);
    const unsigned mask = __ballot_sync(0xffffffffu, in);
    if (lane == 0) warp_n[warp] = __popc(mask);
    __syncthreads();
    int before = base, all = base;
    for (int w = 0; w < 32; w++) {
      if (w < warp) before += warp_n[w];
      all += warp_n[w];
    }
    if (in) {
      rows[before + __popc(mask & ((1u << lane) - 1u))] = (int)r;
    } else if (r < N) {
      loss[r] = 0.f;
      lse[r] = 0.f;
    }
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// dst[i] = src[row i] for i < n (row i = rows[off + i] of the plan, or i itself without one; the row is zero where
// it does not count), rows up to the next multiple of 64 zeroed. One warp per row.
__global__ void __launch_bounds__(256)
    vocab_pack_kernel(const __nv_bfloat16* __restrict__ src, long ld, long D, Answers a, const int* __restrict__ rows,
                      const int* __restrict__ count, long off, long n, __nv_bfloat16* __restrict__ dst, long ldd) {
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long have = count ? min(n, max(0L, (long)*count - off)) : n;
  if (i >= (have + 63) / 64 * 64) return;
  bool in = i < have;
  long r = i;
  if (in) {
    if (rows)
      r = rows[off + i];
    else if (a.ids)
      in = row_counts(a, r);
  }
  __nv_bfloat16* d = dst + i * ldd;
  const __nv_bfloat16* s = src + r * ld;
  if (((uintptr_t)src & 15) == 0 && ld % 8 == 0 && D % 8 == 0) {
    for (long c = lane * 8; c < D; c += 256)
      *reinterpret_cast<uint4*>(d + c) = in ? *reinterpret_cast<const uint4*>(s + c) : make_uint4(0, 0, 0, 0);
  } else {
    for (long c = lane; c < D; c += 32) d[c] = in ? s[c] : __float2bfloat16_rn(0.f);
  }
}

// bias2 = bias / T in log2 units, finite values kept finite (the type's lowest value may stand for a mask).
__global__ void __launch_bounds__(256)
    vocab_bias_kernel(const __nv_bfloat16* __restrict__ bias, long V, long Vp, float scale2, float* __restrict__ out) {
  const long v = (long)blockIdx.x * 256 + threadIdx.x;
  if (v >= Vp) return;
  float b = v < V ? __bfloat162float(bias[v]) : 0.f;
  if (isfinite(b)) b = fminf(fmaxf(b * scale2, -1e38f), 1e38f);
  out[v] = b;
}

__device__ __forceinline__ float block_max(float v, float* scr) {  // 128 threads
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) scr[threadIdx.x >> 5] = v;
  __syncthreads();
  v = fmaxf(fmaxf(scr[0], scr[1]), fmaxf(scr[2], scr[3]));
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* scr) {  // 128 threads, a fixed order
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) scr[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (scr[0] + scr[1]) + (scr[2] + scr[3]);
  __syncthreads();
  return v;
}

// One block per row of the piece: the answer's logits (K products of length D with gathered rows of W: exact to
// f32, which the terms in f16 are not), the row's lse from its segments, the loss, and what the gradient needs:
// info[i] = (lse in log2 units, scale / T), uk[i][k] = u of entry k in log2 units, pk[i][k] its probability.
__global__ void __launch_bounds__(128)
    vocab_rows_kernel(const __nv_bfloat16* __restrict__ x, long ldx, const __nv_bfloat16* __restrict__ w, long ldw,
                      const float* __restrict__ bias2, long V, long D, Answers a, float scale2, float inv_t,
                      const float* __restrict__ row_scale, const int* __restrict__ rows, const int* __restrict__ count,
                      long off, const float2* __restrict__ stat, long ld_stat, float* __restrict__ loss,
                      float* __restrict__ lse, float2* __restrict__ info, float* __restrict__ uk,
                      float* __restrict__ pk) {
  __shared__ float scr[4];
  const long i = blockIdx.x;
  if (count && off + i >= *count) return;
  const long r = rows ? rows[off + i] : off + i;
  const long K = a.K;
  const int* ids = a.ids + r * K;
  if (!rows && !row_counts(a, r)) {
    if (threadIdx.x == 0) {
      loss[r] = 0.f;
      lse[r] = 0.f;
      if (info) info[i] = make_float2(0.f, 0.f);
    }
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // lse2 = max + log2 sum over the segments
  const float2* sr = stat + i * ld_stat;
  float mx = -INFINITY;
  for (long q = threadIdx.x; q < ld_stat; q += 128) mx = fmaxf(mx, sr[q].x);
  mx = block_max(mx, scr);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float s = 0.f;
  for (long q = threadIdx.x; q < ld_stat; q += 128) {
    const float2 f = sr[q];
    s += f.x == -INFINITY ? f.y : f.y * exp2f(f.x - ref);  // an empty segment's sum is 0 (or NaN)
  }
  s = block_sum(s, scr);
  float lse2 = ref + log2f(s);
  // the answer's distribution
  float top = -INFINITY, tot = 1.f;
  bool bad = false;
  const float tscale = inv_t * kLog2e;
  if (a.teacher) {
    for (long k = threadIdx.x; k < K; k += 128)
      if (ids[k] >= 0) top = fmaxf(top, a.teacher[r * K + k]);
    top = block_max(top, scr);
    tot = 0.f;
    for (long k = threadIdx.x; k < K; k += 128)
      if (ids[k] >= 0) tot += exp2f((a.teacher[r * K + k] - top) * tscale);
    tot = block_sum(tot, scr);
  }
  const float log_tot = log2f(tot);
  // sum_k p_k (log2 p_k - u_k), entry k on warp k mod 4
  const __nv_bfloat16* xr = x + i * ldx;
  const bool vec = ((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && ldx % 8 == 0 && ldw % 8 == 0;
  float acc = 0.f;
  for (long k = warp; k < K; k += 4) {
    const int id = ids[k];
    float p = 0.f, u = 0.f, logp = 0.f;
    if (id >= 0) {
      p = 1.f;
      if (a.teacher) {
        logp = (a.teacher[r * K + k] - top) * tscale - log_tot;
        p = exp2f(logp);
      }
      if (id >= V) {
        bad = true;
      } else {
        const __nv_bfloat16* wr = w + (long)id * ldw;
        float d = 0.f;
        long c = 0;
        if (vec) {
          const long Dv = D / 8 * 8;
#pragma unroll 4
          for (c = lane * 8; c < Dv; c += 256) {
            const uint4 xv = *reinterpret_cast<const uint4*>(xr + c), wv = __ldg(reinterpret_cast<const uint4*>(wr + c));
            const __nv_bfloat162 *xh = reinterpret_cast<const __nv_bfloat162*>(&xv),
                                 *wh = reinterpret_cast<const __nv_bfloat162*>(&wv);
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 f = __bfloat1622float2(xh[j]), g = __bfloat1622float2(wh[j]);
              d = __fmaf_rn(f.x, g.x, d);
              d = __fmaf_rn(f.y, g.y, d);
            }
          }
          c = Dv;
        }
        for (c += lane; c < D; c += 32) d = __fmaf_rn(__bfloat162float(xr[c]), __bfloat162float(wr[c]), d);
#pragma unroll
        for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        u = __fmaf_rn(d, scale2, bias2 ? bias2[id] : 0.f);
        if (p > 0.f) acc = __fmaf_rn(p, logp - u, acc);
        else if (isnan(p)) acc = p;
      }
    }
    if (lane == 0 && info) {
      uk[i * K + k] = u;
      pk[i * K + k] = p;
    }
  }
  acc = block_sum(lane == 0 ? acc : 0.f, scr);
  if (block_sum(bad ? 1.f : 0.f, scr) > 0.f) acc = lse2 = NAN;  // an index past the vocabulary: seen in the loss
  if (threadIdx.x == 0) {
    loss[r] = (acc + lse2) * kLn2;
    lse[r] = lse2 * kLn2;
    if (info) info[i] = make_float2(lse2, (row_scale ? row_scale[r] : 1.f) * inv_t);
  }
}

// The f16 terms of a 64-row x 256-column tile become dz in place (bf16): t 2^(max - lse - 15) scale, and at the
// answer's columns scale (2^(u - lse) - sum p) from the f32 logits. A warp walks the rows, a lane owns 8 columns;
// which rows have an answer in the tile is found first, so that the others pay one flag. With `part` each lane's
// column sums (of the unrounded values) go to part[row tile][V] for dbias. Rows from the count to the next
// multiple of 64 are zeroed (the weight-gradient product reads whole k-blocks of rows).
__global__ void __launch_bounds__(256)
    vocab_dz_kernel(void* __restrict__ terms, long ld, long V, Answers a, const int* __restrict__ rows,
                    const int* __restrict__ count, long off, long n, const float2* __restrict__ info,
                    const float* __restrict__ uk, const float* __restrict__ pk, const float2* __restrict__ stat,
                    long ld_stat, int seg, float* __restrict__ part) {
  __shared__ int hit[64];
  __shared__ float fold[8][256];
  const long have = count ? min(n, max(0L, (long)*count - off)) : n;
  const long r0 = (long)blockIdx.y * 64, c0 = (long)blockIdx.x * 256;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long c = c0 + lane * 8;
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; j++) sum[j] = 0.f;
  if (r0 < have) {
    const int nr = (int)min(64L, have - r0);
    if (threadIdx.x < 64) hit[threadIdx.x] = 0;
    __syncthreads();
    for (long q = threadIdx.x; q < nr * a.K; q += 256) {
      const long i = r0 + q / a.K, k = q - q / a.K * a.K;
      const int id = a.ids[(rows ? (long)rows[off + i] : off + i) * a.K + k];
      if (id >= c0 && id < c0 + 256) hit[i - r0] = 1;
    }
    __syncthreads();
    if (c < V) {  // V's pad up to a multiple of 8 lies inside ld
#pragma unroll 4
      for (int q = warp; q < 64; q += 8) {
        const long i = r0 + q;
        uint4* at = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(terms) + i * ld + c);
        float v[8];
        if (q < nr) {
          const float2 f = info[i];  // (lse2, scale)
          const uint4 raw = *at;
          const __half2* h = reinterpret_cast<const __half2*>(&raw);
          if (f.y == 0.f) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.f;
          } else {
            const float m = stat[i * ld_stat + c / seg].x;
            const float k = m == -INFINITY ? 0.f : exp2f(m - f.x - 15.f) * f.y;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 t = __half22float2(h[j]);
              v[2 * j] = t.x * k;
              v[2 * j + 1] = t.y * k;
            }
            if (hit[q]) {
              const int* ids = a.ids + (rows ? (long)rows[off + i] : off + i) * a.K;
              for (long e = 0; e < a.K; e++) {
                const long d = (long)ids[e] - c;
                if (d < 0 || d >= 8) continue;
                float p = 0.f;  // entries that name the same column add up
                for (long g = 0; g < a.K; g++)
                  if (ids[g] == ids[e]) p += pk[i * a.K + g];
                const float val = (exp2f(uk[i * a.K + e] - f.x) - p) * f.y;
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = j == (int)d ? val : v[j];
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 8; j++) sum[j] += v[j];
        } else {
          if (i >= (have + 63) / 64 * 64) continue;
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = 0.f;
        }
        uint4 o;
        uint32_t* u = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          u[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *at = o;
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; j++) fold[warp][lane * 8 + j] = sum[j];
  __syncthreads();
  const long cc = c0 + threadIdx.x;
  if (cc < V) {
    float t = fold[0][threadIdx.x];
#pragma unroll
    for (int q = 1; q < 8; q++) t += fold[q][threadIdx.x];
    part[(long)blockIdx.y * V + cc] = t;
  }
}

// sum (+)= the row tiles' column sums; on the last piece dbias = sum (f32 or bf16).
__global__ void __launch_bounds__(256)
    vocab_dbias_kernel(const float* __restrict__ part, int tiles, long V, float* __restrict__ acc, int first, int last,
                       int f32, void* __restrict__ dbias) {
  const long v = (long)blockIdx.x * 256 + threadIdx.x;
  if (v >= V) return;
  float s = first ? 0.f : acc[v];
#pragma unroll 4
  for (int q = 0; q < tiles; q++) s += part[(long)q * V + v];
  if (!last)
    acc[v] = s;
  else if (f32)
    reinterpret_cast<float*>(dbias)[v] = s;
  else
    reinterpret_cast<__nv_bfloat16*>(dbias)[v] = __float2bfloat16_rn(s);
}

// dx row rows[off + i] = row i of `src`, i < the rows that count: summed over `splits` f32 slices or copied from
// bf16. One warp per row.
__global__ void __launch_bounds__(256)
    vocab_dx_kernel(const void* __restrict__ src, long lds, long slice, int splits, const int* __restrict__ rows,
                    const int* __restrict__ count, long off, long n, long D, __nv_bfloat16* __restrict__ dx, long lddx) {
  const long i = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long have = count ? min(n, max(0L, (long)*count - off)) : n;
  const bool vec = ((uintptr_t)dx & 15) == 0 && lddx % 8 == 0 && D % 8 == 0;
  if (i >= have) return;
  const long r = rows ? rows[off + i] : off + i;
  __nv_bfloat16* d = dx + r * lddx;
  if (splits > 0) {
    const float* s = reinterpret_cast<const float*>(src) + i * lds;
    if (vec) {
      for (long c = lane * 8; c < D; c += 256) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int z = 0; z < splits; z++) {
          const float4 p = *reinterpret_cast<const float4*>(s + z * slice + c),
                       q = *reinterpret_cast<const float4*>(s + z * slice + c + 4);
          v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w, v[4] += q.x, v[5] += q.y, v[6] += q.z, v[7] += q.w;
        }
        uint4 o;
        uint32_t* u = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          u[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(d + c) = o;
      }
    } else {
      for (long c = lane; c < D; c += 32) {
        float v = 0.f;
        for (int z = 0; z < splits; z++) v += s[z * slice + c];
        d[c] = __float2bfloat16_rn(v);
      }
    }
  } else {
    const __nv_bfloat16* s = reinterpret_cast<const __nv_bfloat16*>(src) + i * lds;
    if (vec) {
      for (long c = lane * 8; c < D; c += 256) *reinterpret_cast<uint4*>(d + c) = *reinterpret_cast<const uint4*>(s + c);
    } else {
      for (long c = lane; c < D; c += 32) d[c] = s[c];
    }
  }
}

// The weight gradient from `splits` f32 slices (and the pieces before, in `acc`): kept in acc, or after the last
// piece written in the caller's type.
__global__ void __launch_bounds__(256)
    vocab_dw_kernel(const float* __restrict__ src, long lds, long slice, int splits, float* __restrict__ acc, int first,
                    int last, long V, long D, int f32, void* __restrict__ dw, long lddw) {
  for (long r = blockIdx.x; r < V; r += gridDim.x)
    for (long c = threadIdx.x; c < D; c += 256) {
      float v = first ? 0.f : acc[r * lds + c];
#pragma unroll 4
      for (int z = 0; z < splits; z++) v += src[z * slice + r * lds + c];
      if (!last)
        acc[r * lds + c] = v;
      else if (f32)
        reinterpret_cast<float*>(dw)[r * lddw + c] = v;
      else
        reinterpret_cast<__nv_bfloat16*>(dw)[r * lddw + c] = __float2bfloat16_rn(v);
    }
}

// ---------------------------------------------------------------------------------------------- host side
// Rows up to which one row tile holds them all: leaving rows out of the products then saves nothing, so no plan is
// made (two launches fewer; the rows without an answer are zeroed instead).
constexpr long kVocabOneTile = 128;
// Bytes of terms that one piece may hold. Fewer pieces mean fewer passes over the f32 weight gradient (each piece
// after the first adds to it: 8 V D bytes).
constexpr size_t kVocabPieceBytes = (size_t)4 << 30;

struct VocabPlan {
  bool grad, compact, pack_x, pack_w, dx_direct;
  long N, V, D, K;
  long Dp;       // row stride of the packed matrices and of dx's
  long ldt;      // row stride of the terms
  int bn;        // column tile of the logits product
  long ld_stat;
  long R;        // rows of a piece
  int pieces;
  int splits, dw_splits;  // slices of the long axes of dx (V) and dW (the rows); 0: one
  size_t bytes;
  // offsets into the workspace
  size_t rows, count, xp, wp, bias2, stat, terms, info, uk, pk, dxs, dws, dwacc, part, dbacc;
};

static size_t carve(size_t& at, size_t bytes) {
  const size_t o = at;
  at += (bytes + 255) / 256 * 256;
  return o;
}

// x_ok, w_ok, dx_ok: the matrix starts at 16 bytes and its row stride is a multiple of 8 (what TMA needs).
static VocabPlan vocab_plan(long N, long V, long D, long K, bool bias, bool grad, bool x_ok, bool w_ok, bool dx_ok,
                            bool dw_bf16, size_t piece_bytes) {
  VocabPlan p{};
  p.grad = grad;
  p.N = N;
  p.V = V;
  p.D = D;
  p.K = K;
  p.compact = N > kVocabOneTile;
  p.pack_x = p.compact || grad || !x_ok;
  p.pack_w = !w_ok;
  p.Dp = round_up(D, 8);
  p.ldt = round_up(V, 64);
  p.bn = V > 148 * 128 ? 256 : 128;
  p.ld_stat = ceil_div(V, p.bn) * 2;
  if (!piece_bytes) piece_bytes = kVocabPieceBytes;
  long R = (long)(piece_bytes / ((size_t)p.ldt * 2)) / 128 * 128;
  if (R < 128) R = 128;
  if (R > round_up(N, 128)) R = round_up(N, 128);
  if (R > (1 << 21)) R = 1 << 21;  // 64-row tiles on a grid's second axis
  p.pieces = (int)ceil_div(N, R);
  p.R = round_up(ceil_div(N, p.pieces), 128);
  p.pieces = (int)ceil_div(N, p.R);
  // Few tiles and a long inner axis are split along it, so that every SM has a part: at least 4 k-blocks of 64.
  auto split = [](long tiles, long inner) {
    long s = 148 / tiles;
    if (s > inner / 256) s = inner / 256;
    return s > 1 ? (int)s : 0;
  };
  if (grad) {
    p.splits = split(ceil_div(p.R, 128) * ceil_div(D, 256), V);
    p.dw_splits = split(ceil_div(V, 128) * ceil_div(D, 256), p.R);
  }
  p.dx_direct = !p.compact && p.splits == 0 && dx_ok;
  size_t at = 0;
  if (p.compact) {
    p.rows = carve(at, (size_t)N * 4);
    p.count = carve(at, 4);
  }
  if (p.pack_x) p.xp = carve(at, (size_t)p.R * p.Dp * 2);
  if (p.pack_w) p.wp = carve(at, (size_t)round_up(V, 64) * p.Dp * 2);
  if (bias) p.bias2 = carve(at, (size_t)round_up(V, 256) * 4);
  p.stat = carve(at, (size_t)p.R * p.ld_stat * 8);
  if (grad) {
    p.terms = carve(at, (size_t)p.R * p.ldt * 2);
    p.info = carve(at, (size_t)p.R * 8);
    p.uk = carve(at, (size_t)p.R * K * 4);
    p.pk = carve(at, (size_t)p.R * K * 4);
    if (p.splits)
      p.dxs = carve(at, (size_t)p.splits * p.R * p.Dp * 4);
    else if (!p.dx_direct)
      p.dxs = carve(at, (size_t)p.R * p.Dp * 2);
    if (p.dw_splits) p.dws = carve(at, (size_t)p.dw_splits * V * p.Dp * 4);
    if (p.pieces > 1 && (dw_bf16 || p.dw_splits)) p.dwacc = carve(at, (size_t)V * p.Dp * 4);
    if (bias) {
      p.part = carve(at, (size_t)(p.R / 64) * V * 4);
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
  Answers a;
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

static int vocab_run(const VocabCall& c) {
  PL_REQUIRE(c.V > 0 && c.D > 0 && c.a.K > 0, PL_ERR_INVALID, "%s: V = %zu, D = %zu, K = %ld", c.what, c.V, c.D, c.a.K);
  PL_REQUIRE(c.N <= (1u << 30) && c.V <= (1u << 30) && c.D <= (1u << 24) && c.a.K <= (1 << 20), PL_ERR_INVALID,
             "%s: N = %zu, V = %zu, D = %zu, K = %ld is too large", c.what, c.N, c.V, c.D, c.a.K);
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
  PL_REQUIRE(c.N == 0 || (c.x && c.a.ids && c.loss && c.lse && (!c.grad || c.dx)), PL_ERR_INVALID, "%s: NULL matrix",
             c.what);
  int rc = require_device();
  if (rc) return rc;
  const long N = (long)c.N, V = (long)c.V, D = (long)c.D, K = c.a.K;
  cudaStream_t st = c.st;
  const size_t wsize = c.dw_f32 ? 4 : 2;
  if (N == 0) {
    if (c.grad) {
      PL_CUDA(cudaMemset2DAsync(c.dw, c.lddw * wsize, 0, c.D * wsize, c.V, st));
      if (c.dbias) PL_CUDA(cudaMemsetAsync(c.dbias, 0, c.V * wsize, st));
    }
    return PL_OK;
  }
  const VocabPlan p = vocab_plan(N, V, D, K, c.bias != nullptr, c.grad, rows16(c.x, c.ldx), rows16(c.w, c.ldw),
                                 c.grad && rows16(c.dx, c.lddx), !c.dw_f32, c.piece_bytes);
  PL_REQUIRE(c.ws && c.ws_bytes >= p.bytes && ((uintptr_t)c.ws & 255) == 0, PL_ERR_INVALID,
             "%s: %zu bytes of workspace (256-byte aligned), %zu needed", c.what, c.ws ? c.ws_bytes : (size_t)0, p.bytes);
  uint8_t* ws = (uint8_t*)c.ws;
  int* rows = p.compact ? (int*)(ws + p.rows) : nullptr;
  int* count = p.compact ? (int*)(ws + p.count) : nullptr;
  const float inv_t = (float)(1.0 / c.temperature);
  const float scale2 = (float)((double)kLog2e / c.temperature);
  float* bias2 = nullptr;
  if (c.bias) {
    bias2 = (float*)(ws + p.bias2);
    const long Vp = round_up(V, 256);
    vocab_bias_kernel<<<(unsigned)(Vp / 256), 256, 0, st>>>((const __nv_bfloat16*)c.bias, V, Vp, scale2, bias2);
    count_launch();
    PL_LAUNCH("vocab_bias_kernel");
  }
  if (p.compact) {
    if (c.grad) PL_CUDA(cudaMemset2DAsync(c.dx, c.lddx * 2, 0, c.D * 2, c.N, st));  // rows that do not count
    vocab_plan_kernel<<<1, 1024, 0, st>>>(c.a, N, rows, count, c.loss, c.lse);
    count_launch();
    PL_LAUNCH("vocab_plan_kernel");
  }
  const __nv_bfloat16* w = (const __nv_bfloat16*)c.w;
  long ldw = (long)c.ldw;
  if (p.pack_w) {
    __nv_bfloat16* wp = (__nv_bfloat16*)(ws + p.wp);
    vocab_pack_kernel<<<(unsigned)ceil_div(round_up(V, 64), 8), 256, 0, st>>>(w, ldw, D, Answers{}, nullptr, nullptr, 0, V,
                                                                             wp, p.Dp);
    count_launch();
    PL_LAUNCH("vocab_pack_kernel");
    w = wp;
    ldw = p.Dp;
  }
  for (int q = 0; q < p.pieces; q++) {
    const long off = (long)q * p.R, n = N - off < p.R ? N - off : p.R;
    const __nv_bfloat16* x = (const __nv_bfloat16*)c.x;  // without a plan there is one piece
    long ldx = (long)c.ldx;
    if (p.pack_x) {
      __nv_bfloat16* xp = (__nv_bfloat16*)(ws + p.xp);
      vocab_pack_kernel<<<(unsigned)ceil_div(round_up(n, 64), 8), 256, 0, st>>>(x, ldx, D, c.a, rows, count, off, n, xp,
                                                                               p.Dp);
      count_launch();
      PL_LAUNCH("vocab_pack_kernel");
      x = xp;
      ldx = p.Dp;
    }
    // logits: statistics of every segment, and the terms
    const Operand X{x, p.pack_x ? p.R : n, D, ldx, 1, 0}, W{w, V, D, ldw, 1, 0};
    EpiArgs e{};
    e.out = c.grad ? ws + p.terms : nullptr;
    e.ldo = p.ldt;
    e.out_rows = (int)(c.grad ? p.R : n);
    e.out_cols = (int)V;
    e.scale2 = scale2;
    e.bias2 = bias2;
    e.stat = (float2*)(ws + p.stat);
    e.ld_stat = p.ld_stat;
    e.dyn_rows = count;
    e.dyn_off = (int)off;
    rc = gemm_launch(p.bn, EPI_VOCAB, false, false, X, W, (int)n, (int)V, (int)D, 1, e, st);
    if (rc) return rc;
    float2* info = c.grad ? (float2*)(ws + p.info) : nullptr;
    float* uk = c.grad ? (float*)(ws + p.uk) : nullptr;
    float* pk = c.grad ? (float*)(ws + p.pk) : nullptr;
    vocab_rows_kernel<<<(unsigned)n, 128, 0, st>>>(x, ldx, w, ldw, bias2, V, D, c.a, scale2, inv_t, c.row_scale, rows,
                                                   count, off, (const float2*)(ws + p.stat), p.ld_stat, c.loss, c.lse,
                                                   info, uk, pk);
    count_launch();
    PL_LAUNCH("vocab_rows_kernel");
    if (!c.grad) continue;
    float* part = c.bias ? (float*)(ws + p.part) : nullptr;
    const long tiles = ceil_div(n, 64);
    vocab_dz_kernel<<<dim3((unsigned)ceil_div(V, 256), (unsigned)tiles), 256, 0, st>>>(
        ws + p.terms, p.ldt, V, c.a, rows, count, off, n, info, uk, pk, (const float2*)(ws + p.stat), p.ld_stat, p.bn / 2,
        part);
    count_launch();
    PL_LAUNCH("vocab_dz_kernel");
    const bool last = q == p.pieces - 1;
    if (c.bias) {
      vocab_dbias_kernel<<<(unsigned)ceil_div(V, 256), 256, 0, st>>>(part, (int)tiles, V, (float*)(ws + p.dbacc), q == 0,
                                                                    last, c.dw_f32, c.dbias);
      count_launch();
      PL_LAUNCH("vocab_dbias_kernel");
    }
    // dx = dz W
    const Operand Z{ws + p.terms, p.R, V, p.ldt, 1, 0};
    {
      EpiArgs g{};
      g.alpha = 1.f;
      g.out_rows = (int)n;
      g.out_cols = (int)D;
      g.dyn_rows = count;
      g.dyn_off = (int)off;
      if (p.dx_direct) {
        g.out = c.dx;
        g.ldo = (long)c.lddx;
      } else {
        g.out = ws + p.dxs;
        g.ldo = p.Dp;
        g.out_bstride = p.R * p.Dp;
      }
      g.k_splits = p.splits;
      const int bn = D > 128 ? 256 : 128;
      rc = gemm_launch(bn, p.splits ? EPI_F32 : EPI_BF16, false, true, Z, W, (int)n, (int)D, (int)V, 1, g, st);
      if (rc) return rc;
    }
    if (!p.dx_direct) {
      vocab_dx_kernel<<<(unsigned)ceil_div(n, 8), 256, 0, st>>>(ws + p.dxs, p.Dp, p.R * p.Dp, p.splits, rows, count, off, n,
                                                               D, (__nv_bfloat16*)c.dx, (long)c.lddx);
      count_launch();
      PL_LAUNCH("vocab_dx_kernel");
    }
    // dW (+)= dz^T x
    {
      EpiArgs g{};
      g.alpha = 1.f;
      g.out_rows = (int)V;
      g.out_cols = (int)D;
      g.dyn_rows = count;
      g.dyn_off = (int)off;
      g.dyn_k = 1;
      // slices, the sum of the pieces so far, or the caller's matrix
      const bool direct = !p.dw_splits && (p.pieces == 1 || c.dw_f32);
      const bool f32 = !direct || c.dw_f32;
      g.out = direct ? c.dw : (void*)(ws + (p.dw_splits ? p.dws : p.dwacc));
      g.ldo = direct ? (long)c.lddw : p.Dp;
      g.out_bstride = V * p.Dp;
      g.k_splits = p.dw_splits;
      g.accum = !p.dw_splits && q > 0;
      const Operand Xk{x, n, D, ldx, 1, 0};
      const Operand Zk{ws + p.terms, n, V, p.ldt, 1, 0};
      const int bn = D > 128 ? 256 : 128;
      rc = gemm_launch(bn, f32 ? EPI_F32 : EPI_BF16, true, true, Zk, Xk, (int)V, (int)D, (int)n, 1, g, st);
      if (rc) return rc;
      if (!direct && (p.dw_splits || last)) {
        float* acc = (float*)(ws + p.dwacc);
        vocab_dw_kernel<<<(unsigned)(V < 148 * 16 ? V : 148 * 16), 256, 0, st>>>(
            p.dw_splits ? (const float*)(ws + p.dws) : acc, p.Dp, V * p.Dp, p.dw_splits ? p.dw_splits : 1, acc,
            !p.dw_splits || q == 0, last, V, D, c.dw_f32, c.dw, (long)c.lddw);
        count_launch();
        PL_LAUNCH("vocab_dw_kernel");
      }
    }
  }
  return PL_OK;
}

}  // namespace pl

extern "C" {

size_t pl_vocab_ws(size_t N, size_t V, size_t D, size_t K, uint8_t bias, uint8_t grad, uint8_t aligned,
                   size_t piece_bytes) {
  if (N == 0 || V == 0 || D == 0 || K == 0) return 0;
  const bool ok = aligned != 0;
  return pl::vocab_plan((long)N, (long)V, (long)D, (long)K, bias != 0, grad != 0, ok, ok, ok, true, piece_bytes).bytes;
}

int pl_vocab_ce_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* target,
                    size_t N, size_t V, size_t D, float* loss, float* lse, void* ws, size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_ce_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.a = pl::Answers{target, nullptr, 1};
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
  c.a = pl::Answers{target, nullptr, 1};
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
  c.a = pl::Answers{ids, teacher, (long)K};
  c.temperature = temperature;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.st = (cudaStream_t)stream;
  if (N > 0 && !teacher) return pl::set_error(PL_ERR_INVALID, "pl_vocab_distill_dev: NULL teacher");
  return pl::vocab_run(c);
}

int pl_vocab_distill_grad_dev(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const int32_t* ids,
                              const float* teacher, size_t K, double temperature, const float* row_scale, size_t N,
                              size_t V, size_t D, float* loss, float* lse, void* dx, size_t lddx, void* dw, size_t lddw,
                              void* dbias, uint8_t dw_f32, size_t piece_bytes, void* ws, size_t ws_bytes, void* stream) {
  pl::VocabCall c{};
  c.what = "pl_vocab_distill_grad_dev";
  c.x = x, c.ldx = ldx, c.w = w, c.ldw = ldw, c.bias = bias;
  c.a = pl::Answers{ids, teacher, (long)K};
  c.temperature = temperature;
  c.row_scale = row_scale;
  c.N = N, c.V = V, c.D = D, c.loss = loss, c.lse = lse, c.ws = ws, c.ws_bytes = ws_bytes;
  c.dx = dx, c.lddx = lddx, c.dw = dw, c.lddw = lddw, c.dbias = dbias, c.dw_f32 = dw_f32, c.piece_bytes = piece_bytes;
  c.grad = true;
  c.st = (cudaStream_t)stream;
  if (N > 0 && !teacher) return pl::set_error(PL_ERR_INVALID, "pl_vocab_distill_grad_dev: NULL teacher");
  return pl::vocab_run(c);
}

}  // extern "C"
