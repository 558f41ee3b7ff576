// The gated delta rule, a matrix memory per head, over packed sequences with its gradient, and one token at a time.
// With a_t = exp(g_t), for every head's state S [dk x dv] (f32), q, k, v, o bf16:
//
//   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),  S_t = a_t S_{t-1} + k_t u_t^T,  o_t = scale S_t^T q_t
//
// Sequences go in chunks of 64 tokens. With G the sums of g in a chunk, D_ij = exp(G_i - G_j) for j <= i, E = diag(exp G),
// F = diag(exp(G_last - G)), N = strictly lower part of K K^T times D, P = lower part of Q K^T times D and S the state before
// the chunk:
//
//   Y = X (V - E K S), X = (I + N diag(beta))^-1, U = diag(beta) Y
//   O = scale (E Q S + P U),  S' = exp(G_last) S + K^T F U
//
// and back, from dO and dS' (the gradient of the state behind the chunk):
//
//   dU = scale P^T dO + F K dS',  dR = X^T diag(beta) dU,  dV = dR
//   dS = exp(G_last) dS' + scale (E Q)^T dO - (E K)^T dR
//   dQ = scale (E dO S^T + (dO U^T * D) K)
//   dK = -E dR S^T + F U dS'^T + scale (dO U^T * D)^T Q - (M + M^T) K,  M = strictly lower part of dR U^T times D
//   dbeta_j = scale sum_i P_ij (dO_i . Y_j) + F_j K_j . (dS' Y_j) - sum_i N_ij (dR_i . Y_j)
//   dg_t = sum over i >= t > j of W_ij, over i >= t of e_i and over j < t of f_j, and exp(G_last) <S, dS'>, with
//          W = scale P * (dO U^T) - N * (dR U^T), e_i = E_i (scale q_i . S dO_i - k_i . S dR_i), f_j = F_j K_j . (dS' U_j)
//
// (up to the resets: what lies on two sides of one has no W, e or f). The sums for dg are taken as those over i >= t of
// W's rows less W's columns: what is left out on both sides is the same number, so the products' errors cancel with it
// (q . dq - v . dv is the same in exact arithmetic, and three times as far off).
//
// X and P depend on q, k, g and beta alone: one kernel makes them for all chunks at once. What is left in the chain over a
// sequence's chunks is a few products with the state, for each 64 columns of v on their own (columns do not mix), and
// what the gradient needs beyond the two chains (S per chunk forward, dS' back) is again one kernel over all chunks.
// f32 operands of products (S, Y, U, dR, X, P) go as two bf16 parts: with one, the states and gradients in f32 would be 2e-3
// off, with two 5e-6.
#include "pl_delta.cuh"
#include "pl_runtime.h"

namespace pl {

// ---------------------------------------------------------------------------------------------- one token
// A block per row, head and 32 VEC columns: the state's tile is read into registers (R rows of every warp), used and written
// once. Bound by HBM: 8 dk dv bytes per row and head.
struct StepArgs {
  DeltaArgs d;
  const float* state;
  float* out;
  __nv_bfloat16* o;
};
template <int VEC>
struct __align__(4 * VEC) Floats {
  float v[VEC];
};
template <int VEC, int R>
__global__ void __launch_bounds__(256) delta_step_kernel(const StepArgs p) {
  grid_wait();
  grid_next();
  constexpr int W = 32 * VEC;
  __shared__ float qk[2][128];
  __shared__ float part[2][8][W];
  const DeltaArgs& a = p.d;
  const long row = blockIdx.x / a.hv;
  const int h = (int)(blockIdx.x % a.hv), hk = h / (a.hv / a.hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.y * W + lane * VEC;
  const bool in = col < a.dv;  // VEC divides dv
  const float* s = p.state + blockIdx.x * (long)a.dk * a.dv;
  Floats<VEC> x[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int i = warp + 8 * r;
    if (i < a.dk && in) {
      x[r] = *reinterpret_cast<const Floats<VEC>*>(s + (long)i * a.dv + col);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) x[r].v[j] = 0.f;
    }
  }
  for (int i = threadIdx.x; i < 256; i += 256) {
    const int c = i & 127;
    const __nv_bfloat16* src = i < 128 ? a.q + row * a.ldq + hk * a.hsq : a.k + row * a.ldk + hk * a.hsk;
    qk[i >> 7][c] = c < a.dk ? __bfloat162float(src[c]) : 0.f;
  }
  const float g = a.g[blockIdx.x], beta = a.beta[blockIdx.x];
  const float decay = g < -104.f ? 0.f : expf(g);
  __syncthreads();
  float dot = 0.f, kq[VEC], qs[VEC];
#pragma unroll
  for (int i = 0; i < 4; i++) dot = __fmaf_rn(qk[0][lane + 32 * i], qk[1][lane + 32 * i], dot);
#pragma unroll
  for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
#pragma unroll
  for (int j = 0; j < VEC; j++) kq[j] = qs[j] = 0.f;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int i = warp + 8 * r;
    const float kk = qk[1][i], qq = qk[0][i];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      x[r].v[j] = decay == 0.f ? 0.f : x[r].v[j] * decay;  // a reset forgets infinities too
      kq[j] = __fmaf_rn(kk, x[r].v[j], kq[j]);
      qs[j] = __fmaf_rn(qq, x[r].v[j], qs[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    part[0][warp][lane * VEC + j] = kq[j];
    part[1][warp][lane * VEC + j] = qs[j];
  }
  __syncthreads();
  float u[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    float ks = 0.f, os = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) {
      ks += part[0][w][lane * VEC + j];
      os += part[1][w][lane * VEC + j];
    }
    u[j] = 0.f;
    if (!in) continue;
    u[j] = beta * (__bfloat162float(a.v[row * a.ldv + h * a.hsv + col + j]) - ks);
    if (warp == 0) p.o[blockIdx.x * (long)a.dv + col + j] = __float2bfloat16_rn(a.scale * __fmaf_rn(dot, u[j], os));
  }
  float* to = p.out + blockIdx.x * (long)a.dk * a.dv;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int i = warp + 8 * r;
    if (i >= a.dk || !in) continue;
    const float kk = qk[1][i];
#pragma unroll
    for (int j = 0; j < VEC; j++) x[r].v[j] = __fmaf_rn(kk, u[j], x[r].v[j]);
    *reinterpret_cast<Floats<VEC>*>(to + (long)i * a.dv + col) = x[r];
  }
}

// ---------------------------------------------------------------------------------------------- X and P of all chunks
// Per slot and value head: X and P, triangular, as two bf16 parts each (in the order X, its second part, P, its second part), and
// since, until, beta of the chunk's tokens.
struct __align__(16) Mats {
  __nv_bfloat16 x[2][kTri], p[2][kTri];
  float since[kC], until[kC], beta[kC];
};

constexpr int kPrepThreads = 128;
template <int DK>
struct PrepShared {
  __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)];
  float at[kC][kC + 4];  // N diag(beta), transposed: [j][i]
  float x[kC][kC + 4];   // its inverse with I
  float y[32][36];
  Decay d;
};
template <int DK>
__global__ void __launch_bounds__(kPrepThreads) delta_prep_kernel(const DeltaArgs a, Mats* __restrict__ mats) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  PrepShared<DK>& sh = *reinterpret_cast<PrepShared<DK>*>(mem);
  constexpr int LD = DK + 8;
  const long slot = blockIdx.x;
  const int kh = blockIdx.y, group = a.hv / a.hk, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long start;
  const int len = slot_chunk(a, slot, start);
  if (len == 0) return;
  copy_tile<DK, LD, kPrepThreads>(sh.k, a.k + start * a.ldk + kh * a.hsk, a.ldk, len, a.dk, a.vec);
  copy_tile<DK, LD, kPrepThreads>(sh.q, a.q + start * a.ldq + kh * a.hsq, a.ldq, len, a.dk, a.vec);
  cp_commit();
  cp_wait<0>();
  __syncthreads();
  float kk[8][4], qk[8][4];  // rows 16 warp.. of K K^T and Q K^T
  zero(kk);
  zero(qk);
  product<false, LD, 0, false, LD, 0, DK / 16>(kk, sh.k, sh.k, warp * 16, 0);
  product<false, LD, 0, false, LD, 0, DK / 16>(qk, sh.q, sh.k, warp * 16, 0);
  for (int e = 0; e < group; e++) {
    const int h = kh * group + e;
    Mats& out = mats[slot * a.hv + h];
    __syncthreads();
    chunk_decay(a, sh.d, start, len, h);
    __syncthreads();
    if (tid < kC) {
      out.since[tid] = sh.d.since[tid];
      out.until[tid] = sh.d.until[tid];
      out.beta[tid] = sh.d.beta[tid];
    }
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = warp * 16 + half * 8 + (lane >> 2), j = t * 8 + (lane & 3) * 2;
        float p[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const float f = j + c <= i ? decay(sh.d, i, j + c) : 0.f;
          p[c] = j + c <= i ? qk[t][half * 2 + c] * f : 0.f;
          sh.at[j + c][i] = j + c < i ? kk[t][half * 2 + c] * f * sh.d.beta[j + c] : 0.f;
        }
        if (j >> 4 <= warp) {
          uint32_t hi, lo;
          split2(p[0], p[1], hi, lo);
          *reinterpret_cast<uint32_t*>(out.p[0] + tri_at(i, j)) = hi;
          *reinterpret_cast<uint32_t*>(out.p[1] + tri_at(i, j)) = lo;
        }
      }
    __syncthreads();
    // the inverse's two diagonal blocks, a column per thread: x_i -= A_ij x_j as soon as x_j is known
    if (tid < 64) {
      const int b = tid & 32, c = tid & 31;
      float x[32];
#pragma unroll
      for (int i = 0; i < 32; i++) x[i] = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < 31; j++)
#pragma unroll
        for (int i = j + 1; i < 32; i++) x[i] = __fmaf_rn(-sh.at[b + j][b + i], x[j], x[i]);
#pragma unroll
      for (int i = 0; i < 32; i++) {
        sh.x[b + i][b + c] = x[i];
        if (b) sh.x[i][b + c] = 0.f;
      }
    }
    __syncthreads();
    {  // the block below: -X22 (A21 X11), eight values per thread
      const int i = tid >> 2, c = (tid & 3) * 8;
      float s[8];
#pragma unroll
      for (int q = 0; q < 8; q++) s[q] = 0.f;
      for (int j = 0; j < 32; j++) {
        const float f = sh.at[j][32 + i];
#pragma unroll
        for (int q = 0; q < 8; q++) s[q] = __fmaf_rn(f, sh.x[j][c + q], s[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; q++) sh.y[i][c + q] = s[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 8; q++) s[q] = 0.f;
      for (int j = 0; j < 32; j++) {
        const float f = -sh.x[32 + i][32 + j];
#pragma unroll
        for (int q = 0; q < 8; q++) s[q] = __fmaf_rn(f, sh.y[j][c + q], s[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; q++) sh.x[32 + i][c + q] = s[q];
    }
    __syncthreads();
    for (int i = tid; i < kC * kC / 2; i += kPrepThreads) {
      const int r = i / (kC / 2), c = i % (kC / 2) * 2;
      uint32_t hi, lo;
      if (c >> 4 > r >> 4) continue;
      split2(sh.x[r][c], sh.x[r][c + 1], hi, lo);
      *reinterpret_cast<uint32_t*>(out.x[0] + tri_at(r, c)) = hi;
      *reinterpret_cast<uint32_t*>(out.x[1] + tri_at(r, c)) = lo;
    }
  }
}

// ---------------------------------------------------------------------------------------------- the chain forward
// What a chain leaves for the gradient, per slot, value head and 64 columns of v, as two bf16 parts one behind the other: a
// state [2][dk][64], rows [2][64][64].
__device__ __forceinline__ long state_at(const DeltaArgs& a, long slot, int h, int slice) {
  return ((slot * a.hv + h) * (a.dvp / 64) + slice) * 2 * a.dk * 64;
}
__device__ __forceinline__ long rows_at(const DeltaArgs& a, long slot, int h, int slice) {
  return ((slot * a.hv + h) * (a.dvp / 64) + slice) * 2 * kC * 64;
}

constexpr int kScanThreads = 512;
constexpr int kRows = kC * kLd;  // a 64 x 64 tile: the distance of its second part
struct ScanArgs {
  DeltaArgs d;
  const Mats* mats;
  const float* state;  // [seqs][hv][dk][dv], or NULL: zero
  __nv_bfloat16* o;    // [n][hv][dv]
  float* final_state;
  __nv_bfloat16 *kept, *y;  // for the gradient: S and Y of every slot; or NULL
};
template <int DK>
struct ScanShared {
  struct In {  // a chunk's inputs, loaded while the chunk before it is worked on
    __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)], v[kC * kLd];
    Mats m;
  } in[2];
  __nv_bfloat16 s[2][DK * kLd];  // the state's columns
  __nv_bfloat16 r[2][kC * kLd], u[2][kC * kLd], w[2][kC * kLd];
};

// Rows that no sequence holds, in front of the first and behind the last: zero. Called by the blocks of those two.
template <typename T>
__device__ __forceinline__ void zero_rows(const DeltaArgs& a, int seq, T* out, long ld, int cols) {
  long from, to;
  seq_bounds(a, seq, from, to);
  for (int side = 0; side < 2; side++) {
    if (side ? seq != a.seqs - 1 : seq != 0) continue;
    const long r0 = side ? to : 0, r1 = side ? a.n : from;
    for (long i = r0 * cols + threadIdx.x; i < r1 * cols; i += blockDim.x) out[i / cols * ld + i % cols] = T(0.f);
  }
}

// A block per sequence, value head and 64 of its columns, 16 warps. They hold the state in registers, 16 rows x 32 columns
// each (dk <= 64: x 16); its two bf16 parts in shared memory are the operand of the next chunk's products. (With one part of
// S, U and P in what goes into o alone, a fifth of the products, o would be 2.5e-3 off instead of 1.7e-3.)
template <int DK>
__global__ void __launch_bounds__(kScanThreads) delta_scan_kernel(const ScanArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  ScanShared<DK>& sh = *reinterpret_cast<ScanShared<DK>*>(mem);
  constexpr int LD = DK + 8, NS = DK / 32;  // n-tiles of a warp's part of the state
  const DeltaArgs& a = p.d;
  const int slice = blockIdx.x, c0 = slice * 64, h = blockIdx.y, seq = blockIdx.z, kh = h / (a.hv / a.hk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
  const int sm = warp % (DK / 16) * 16, sn = warp / (DK / 16) * NS * 8;
  long from, to;
  seq_bounds(a, seq, from, to);
  const long slot0 = from / kC + seq;
  auto load = [&](long c) {
    const long start = from + c * kC;
    const int len = (int)(to - start < kC ? to - start : kC);
    auto& in = sh.in[c & 1];
    copy_tile<DK, LD, kScanThreads>(in.k, a.k + start * a.ldk + kh * a.hsk, a.ldk, len, a.dk, a.vec);
    copy_flat<kScanThreads>(&in.m, p.mats + (slot0 + c) * a.hv + h, sizeof(Mats));
    copy_tile<64, kLd, kScanThreads>(in.v, a.v + start * a.ldv + h * a.hsv + c0, a.ldv, len, cols, a.vec);
    copy_tile<DK, LD, kScanThreads>(in.q, a.q + start * a.ldq + kh * a.hsq, a.ldq, len, a.dk, a.vec);
    cp_commit();
  };
  const long chunks = (to - from + kC - 1) / kC;
  if (chunks) load(0);
  zero_rows(a, seq, p.o + (long)h * a.dv + c0, (long)a.hv * a.dv, cols);
  float s[NS][4];
  const long sbase = ((long)seq * a.hv + h) * a.dk * a.dv + c0;
#pragma unroll
  for (int t = 0; t < NS; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = sm + (lane >> 2) + (e >> 1) * 8, j = sn + t * 8 + (lane & 3) * 2 + (e & 1);
      s[t][e] = p.state && i < a.dk && j < cols ? p.state[sbase + (long)i * a.dv + j] : 0.f;
    }
  for (long c = 0; c < chunks; c++) {
    const long start = from + c * kC, slot = slot0 + c;
    const int len = (int)(to - start < kC ? to - start : kC);
    const auto& in = sh.in[c & 1];
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
      for (int half = 0; half < 2; half++)
        put2<kLd>(sh.s[0], sh.s[1], sm + (lane >> 2) + half * 8, sn + t * 8 + (lane & 3) * 2, s[t][half * 2],
                  s[t][half * 2 + 1]);
    cp_wait<0>();
    __syncthreads();
    if (c + 1 < chunks) load(c + 1);
    if (p.kept)
#pragma unroll
      for (int part = 0; part < 2; part++)
        tile_out<kScanThreads>(p.kept + state_at(a, slot, h, slice) + part * a.dk * 64, sh.s[part], a.dk);
    // warps 0 to 7: V - E K S; warps 8 to 15: E Q S; 16 rows x 32 columns each
    const int m0 = (warp & 3) * 16, n0 = (warp >> 2 & 1) * 32, i0 = m0 + (lane >> 2);
    float acc[4][4];
    zero(acc);
    product<false, LD, 0, true, kLd, DK * kLd, DK / 16>(acc, warp < 8 ? in.k : in.q, sh.s[0], m0, n0);
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int i = i0 + half * 8;
      const float f = in.m.since[i];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const int j = n0 + t * 8 + (lane & 3) * 2;
        float x = f == 0.f ? 0.f : f * acc[t][half * 2], y = f == 0.f ? 0.f : f * acc[t][half * 2 + 1];
        if (warp < 8) {
          const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(in.v + i * kLd + j);
          put2<kLd>(sh.r[0], sh.r[1], i, j, __low2float(v) - x, __high2float(v) - y);
        } else {
          acc[t][half * 2] = x;
          acc[t][half * 2 + 1] = y;
        }
      }
    }
    __syncthreads();
    {  // Y = X R, 16 rows x 16 columns of every warp
      const int y0 = (warp >> 2) * 16;
      float y[2][4];
      zero(y);
      tri_product<false, true, kLd, kRows>(y, in.m.x[0], sh.r[0], warp & 3, y0);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8;
        const float b = in.m.beta[i], f = in.m.until[i];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const int j = y0 + t * 8 + (lane & 3) * 2;
          const float y1 = y[t][half * 2], y2 = y[t][half * 2 + 1];
          if (p.y) {
            uint32_t hi, lo;
            split2(y1, y2, hi, lo);
            __nv_bfloat16* to_y = p.y + rows_at(a, slot, h, slice) + i * 64 + j;
            *reinterpret_cast<uint32_t*>(to_y) = hi;
            *reinterpret_cast<uint32_t*>(to_y + kC * 64) = lo;
          }
          put2<kLd>(sh.u[0], sh.u[1], i, j, b * y1, b * y2);
          put2<kLd>(sh.w[0], sh.w[1], i, j, f * b * y1, f * b * y2);
        }
      }
    }
    __syncthreads();
    const float keep = in.m.since[kC - 1];
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[t][e] = keep == 0.f ? 0.f : keep * s[t][e];
    product<true, LD, 0, true, kLd, kRows, 4>(s, in.k, sh.w[0], sm, sn);
    if (warp >= 8) {
      tri_product<false, true, kLd, kRows>(acc, in.m.p[0], sh.u[0], warp & 3, n0);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8;
        if (i >= len) continue;
        __nv_bfloat16* o = p.o + (start + i) * a.hv * a.dv + (long)h * a.dv + c0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const int j = n0 + t * 8 + (lane & 3) * 2;
          const float x = a.scale * acc[t][half * 2], y = a.scale * acc[t][half * 2 + 1];
          if (a.dv % 2 == 0 && j + 1 < cols) {
            *reinterpret_cast<__nv_bfloat162*>(o + j) = __floats2bfloat162_rn(x, y);
          } else {
            if (j < cols) o[j] = __float2bfloat16_rn(x);
            if (j + 1 < cols) o[j + 1] = __float2bfloat16_rn(y);
          }
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NS; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = sm + (lane >> 2) + (e >> 1) * 8, j = sn + t * 8 + (lane & 3) * 2 + (e & 1);
      if (i < a.dk && j < cols) p.final_state[sbase + (long)i * a.dv + j] = s[t][e];
    }
}

// ---------------------------------------------------------------------------------------------- the chain back
struct BackArgs {
  DeltaArgs d;
  const Mats* mats;
  const __nv_bfloat16* dout;  // [n][hv][dv], strides below
  long ldo, hso;
  bool vec_o;
  const float* dfinal;        // [seqs][hv][dk][dv], or NULL: zero
  __nv_bfloat16* dv;          // [n][hv][dv]
  float* dstate;              // or NULL
  __nv_bfloat16 *ds, *dr;     // dS' and dR of every slot
};
template <int DK>
struct BackShared {
  struct In {
    __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)], o[kC * kLd];
    Mats m;
  } in[2];
  __nv_bfloat16 s[2][DK * kLd];
  __nv_bfloat16 u[2][kC * kLd], r[2][kC * kLd], w[2][kC * kLd];
};
// As the chain forward, from the last chunk to the first.
template <int DK>
__global__ void __launch_bounds__(kScanThreads) delta_back_kernel(const BackArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  BackShared<DK>& sh = *reinterpret_cast<BackShared<DK>*>(mem);
  constexpr int LD = DK + 8, NS = DK / 32;
  const DeltaArgs& a = p.d;
  const int slice = blockIdx.x, c0 = slice * 64, h = blockIdx.y, seq = blockIdx.z, kh = h / (a.hv / a.hk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
  const int sm = warp % (DK / 16) * 16, sn = warp / (DK / 16) * NS * 8;
  long from, to;
  seq_bounds(a, seq, from, to);
  const long slot0 = from / kC + seq, chunks = (to - from + kC - 1) / kC;
  auto load = [&](long c) {
    const long start = from + c * kC;
    const int len = (int)(to - start < kC ? to - start : kC);
    auto& in = sh.in[c & 1];
    copy_tile<DK, LD, kScanThreads>(in.k, a.k + start * a.ldk + kh * a.hsk, a.ldk, len, a.dk, a.vec);
    copy_flat<kScanThreads>(&in.m, p.mats + (slot0 + c) * a.hv + h, sizeof(Mats));
    copy_tile<64, kLd, kScanThreads>(in.o, p.dout + start * p.ldo + h * p.hso + c0, p.ldo, len, cols, p.vec_o);
    copy_tile<DK, LD, kScanThreads>(in.q, a.q + start * a.ldq + kh * a.hsq, a.ldq, len, a.dk, a.vec);
    cp_commit();
  };
  if (chunks) load(chunks - 1);
  zero_rows(a, seq, p.dv + (long)h * a.dv + c0, (long)a.hv * a.dv, cols);
  float s[NS][4];
  const long sbase = ((long)seq * a.hv + h) * a.dk * a.dv + c0;
#pragma unroll
  for (int t = 0; t < NS; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = sm + (lane >> 2) + (e >> 1) * 8, j = sn + t * 8 + (lane & 3) * 2 + (e & 1);
      s[t][e] = p.dfinal && i < a.dk && j < cols ? p.dfinal[sbase + (long)i * a.dv + j] : 0.f;
    }
  const int mt = warp & 3, m0 = mt * 16, n0 = (warp >> 2) * 16, i0 = m0 + (lane >> 2);  // 16 x 16 of a 64 x 64 tile
  for (long c = chunks - 1; c >= 0; c--) {
    const long start = from + c * kC, slot = slot0 + c;
    const int len = (int)(to - start < kC ? to - start : kC);
    const auto& in = sh.in[c & 1];
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
      for (int half = 0; half < 2; half++)
        put2<kLd>(sh.s[0], sh.s[1], sm + (lane >> 2) + half * 8, sn + t * 8 + (lane & 3) * 2, s[t][half * 2],
                  s[t][half * 2 + 1]);
    cp_wait<0>();
    __syncthreads();
    if (c > 0) load(c - 1);
#pragma unroll
    for (int part = 0; part < 2; part++)
      tile_out<kScanThreads>(p.ds + state_at(a, slot, h, slice) + part * a.dk * 64, sh.s[part], a.dk);
    {  // diag(beta) dU = beta (F K dS' + scale P^T dO)
      float x[2][4], y[2][4];
      zero(x);
      zero(y);
      product<false, LD, 0, true, kLd, DK * kLd, DK / 16>(x, in.k, sh.s[0], m0, n0);
      tri_product<true, true, kLd, 0>(y, in.m.p[0], in.o, mt, n0);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8;
        const float b = in.m.beta[i], f = in.m.until[i];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          float z[2];
#pragma unroll
          for (int e = 0; e < 2; e++)
            z[e] = b * ((f == 0.f ? 0.f : f * x[t][half * 2 + e]) + a.scale * y[t][half * 2 + e]);
          put2<kLd>(sh.u[0], sh.u[1], i, n0 + t * 8 + (lane & 3) * 2, z[0], z[1]);
        }
      }
    }
    // scale E dO, the operand of Q's part
    for (int i = tid; i < kC * 32; i += kScanThreads) {
      const int r = i >> 5, cc = (i & 31) * 2;
      const float f = a.scale * in.m.since[r];
      const __nv_bfloat162 o = *reinterpret_cast<const __nv_bfloat162*>(in.o + r * kLd + cc);
      put2<kLd>(sh.w[0], sh.w[1], r, cc, f == 0.f ? 0.f : f * __low2float(o), f == 0.f ? 0.f : f * __high2float(o));
    }
    __syncthreads();
    {  // dR = X^T (beta dU)
      float x[2][4];
      zero(x);
      tri_product<true, true, kLd, kRows>(x, in.m.x[0], sh.u[0], mt, n0);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8;
        const float f = -in.m.since[i];
        __nv_bfloat16* dv = p.dv + (start + i) * a.hv * a.dv + (long)h * a.dv + c0;
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const int j = n0 + t * 8 + (lane & 3) * 2;
          const float y0 = x[t][half * 2], y1 = x[t][half * 2 + 1];
          uint32_t hi, lo;
          split2(y0, y1, hi, lo);
          __nv_bfloat16* to_r = p.dr + rows_at(a, slot, h, slice) + i * 64 + j;
          *reinterpret_cast<uint32_t*>(to_r) = hi;
          *reinterpret_cast<uint32_t*>(to_r + kC * 64) = lo;
          if (i < len) {
            if (a.dv % 2 == 0 && j + 1 < cols) {
              *reinterpret_cast<uint32_t*>(dv + j) = hi;
            } else {
              if (j < cols) dv[j] = __float2bfloat16_rn(y0);
              if (j + 1 < cols) dv[j + 1] = __float2bfloat16_rn(y1);
            }
          }
          put2<kLd>(sh.r[0], sh.r[1], i, j, f == 0.f ? 0.f : f * y0, f == 0.f ? 0.f : f * y1);
        }
      }
    }
    const float keep = in.m.since[kC - 1];
#pragma unroll
    for (int t = 0; t < NS; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[t][e] = keep == 0.f ? 0.f : keep * s[t][e];
    product<true, LD, 0, true, kLd, kRows, 4>(s, in.q, sh.w[0], sm, sn);
    __syncthreads();
    product<true, LD, 0, true, kLd, kRows, 4>(s, in.k, sh.r[0], sm, sn);
  }
  if (!p.dstate) return;
#pragma unroll
  for (int t = 0; t < NS; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = sm + (lane >> 2) + (e >> 1) * 8, j = sn + t * 8 + (lane & 3) * 2 + (e & 1);
      if (i < a.dk && j < cols) p.dstate[sbase + (long)i * a.dv + j] = s[t][e];
    }
}

// ---------------------------------------------------------------------------------------------- the other gradients
struct GradArgs {
  DeltaArgs d;
  const __nv_bfloat16* dout;
  long ldo, hso;
  bool vec_o;
  const __nv_bfloat16 *kept, *y, *ds, *dr;
  __nv_bfloat16 *dq, *dk;  // [n][hk][dk]
  float *dg, *dbeta;       // [n][hv]
};
template <int DK>
struct GradShared {
  __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)];
  __nv_bfloat16 o[2][kC * kLd], r[2][2][kC * kLd];  // by turns: the next step's are on their way
  __nv_bfloat16 s[2][DK * kLd], ds[2][DK * kLd], y[2][kC * kLd];
  __nv_bfloat16 p[2][kC * kLd], m[2][kC * kLd];     // scale dO U^T * D, -M
  float row[4][kC], col[4][kC], krow[4][kC], sum[16];
  Decay d;
};
// A block per chunk and key head, 16 warps: its value heads one after the other, so that what they add to dq and dk stays in
// registers and is added in their order; of each, 64 columns of v after the other (a step). A step's loads are under
// way during the one before it.
template <int DK>
__global__ void __launch_bounds__(kScanThreads) delta_grad_kernel(const GradArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  GradShared<DK>& sh = *reinterpret_cast<GradShared<DK>*>(mem);
  constexpr int LD = DK + 8, NK = DK / 32;  // n-tiles of a warp's quarter of dk
  const DeltaArgs& a = p.d;
  const long slot = blockIdx.x;
  const int kh = blockIdx.y, group = a.hv / a.hk, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long start;
  const int len = slot_chunk(a, slot, start);
  if (len == 0) return;
  const int slices = a.dvp / 64, steps = group * slices;
  auto load_a = [&](int t) {  // S, dO, dR
    const int h = kh * group + t / slices, slice = t % slices, c0 = slice * 64;
    const int cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
    copy_tile<64, kLd, kScanThreads>(sh.o[t & 1], p.dout + start * p.ldo + h * p.hso + c0, p.ldo, len, cols, p.vec_o);
#pragma unroll
    for (int part = 0; part < 2; part++) {
      tile_in<kScanThreads>(sh.s[part], p.kept + state_at(a, slot, h, slice) + part * a.dk * 64, a.dk);
      tile_in<kScanThreads>(sh.r[t & 1][part], p.dr + rows_at(a, slot, h, slice) + part * kC * 64, kC);
    }
    cp_commit();
  };
  auto load_b = [&](int t) {  // dS', Y
    const int h = kh * group + t / slices, slice = t % slices;
#pragma unroll
    for (int part = 0; part < 2; part++) {
      tile_in<kScanThreads>(sh.ds[part], p.ds + state_at(a, slot, h, slice) + part * a.dk * 64, a.dk);
      tile_in<kScanThreads>(sh.y[part], p.y + rows_at(a, slot, h, slice) + part * kC * 64, kC);
    }
    cp_commit();
  };
  copy_tile<DK, LD, kScanThreads>(sh.k, a.k + start * a.ldk + kh * a.hsk, a.ldk, len, a.dk, a.vec);
  copy_tile<DK, LD, kScanThreads>(sh.q, a.q + start * a.ldq + kh * a.hsq, a.ldq, len, a.dk, a.vec);
  load_a(0);
  load_b(0);
  // the states' rows behind dk stay zero
  for (int i = a.dk * kLd + tid; i < DK * kLd; i += kScanThreads)
    sh.s[0][i] = sh.s[1][i] = sh.ds[0][i] = sh.ds[1][i] = __float2bfloat16_rn(0.f);
  const int wr = warp & 3, wc = warp >> 2, m0 = wr * 16, i0 = m0 + (lane >> 2);
  const int n0 = wc * 16, d0 = wc * (DK / 4);  // this warp's columns of a 64 x 64 tile, of a 64 x dk tile
  float dq[NK][4], dk[NK][4], oy[2][4], ry[2][4], qrow[2], krow[2], inner = 0.f;
  zero(dq);
  zero(dk);
  for (int t = 0; t < steps; t++) {
    const int h = kh * group + t / slices;
    const __nv_bfloat16* o = sh.o[t & 1];
    const __nv_bfloat16* r = sh.r[t & 1][0];
    if (t % slices == 0) {
      chunk_decay(a, sh.d, start, len, h);
      zero(oy);
      zero(ry);
      inner = qrow[0] = qrow[1] = krow[0] = krow[1] = 0.f;
    }
    cp_wait<1>();
    __syncthreads();
    float x[NK][4];
    zero(x);
    product<false, kLd, 0, false, kLd, DK * kLd, 4>(x, o, sh.s[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // scale E dO S^T, and what it adds to e_i
      const int i = i0 + half * 8;
      const float f = sh.d.since[i] * a.scale;
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const __nv_bfloat162 q = *reinterpret_cast<const __nv_bfloat162*>(sh.q + i * LD + d0 + n * 8 + (lane & 3) * 2);
        const float v0 = f == 0.f ? 0.f : f * x[n][half * 2], v1 = f == 0.f ? 0.f : f * x[n][half * 2 + 1];
        qrow[half] = __fmaf_rn(__low2float(q), v0, __fmaf_rn(__high2float(q), v1, qrow[half]));
        dq[n][half * 2] += v0;
        dq[n][half * 2 + 1] += v1;
      }
    }
    zero(x);
    product<false, kLd, kRows, false, kLd, DK * kLd, 4>(x, r, sh.s[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // -E dR S^T
      const int i = i0 + half * 8;
      const float f = -sh.d.since[i];
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const __nv_bfloat162 k = *reinterpret_cast<const __nv_bfloat162*>(sh.k + i * LD + d0 + n * 8 + (lane & 3) * 2);
        const float v0 = f == 0.f ? 0.f : f * x[n][half * 2], v1 = f == 0.f ? 0.f : f * x[n][half * 2 + 1];
        qrow[half] = __fmaf_rn(__low2float(k), v0, __fmaf_rn(__high2float(k), v1, qrow[half]));
        dk[n][half * 2] += v0;
        dk[n][half * 2 + 1] += v1;
      }
    }
    cp_wait<0>();
    __syncthreads();
    for (int i = tid; i < DK * 32; i += kScanThreads) {  // <S, dS'>
      const int at = (i >> 5) * kLd + (i & 31) * 2;
      auto two = [&](const __nv_bfloat16* hi, const __nv_bfloat16* lo) {
        const __nv_bfloat162 h2 = *reinterpret_cast<const __nv_bfloat162*>(hi + at), l2 = *reinterpret_cast<const __nv_bfloat162*>(lo + at);
        return make_float2(__low2float(h2) + __low2float(l2), __high2float(h2) + __high2float(l2));
      };
      const float2 u = two(sh.s[0], sh.s[1]), v = two(sh.ds[0], sh.ds[1]);
      inner = __fmaf_rn(u.x, v.x, __fmaf_rn(u.y, v.y, inner));
    }
    __syncthreads();
    if (t + 1 < steps) load_a(t + 1);
    zero(x);
    product<false, kLd, kRows, false, kLd, DK * kLd, 4>(x, sh.y[0], sh.ds[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // F U dS'^T, and K_i . (dS' Y_i)
      const int i = i0 + half * 8;
      const float f = sh.d.until[i], b = sh.d.beta[i];
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const __nv_bfloat162 k = *reinterpret_cast<const __nv_bfloat162*>(sh.k + i * LD + d0 + n * 8 + (lane & 3) * 2);
        const float v0 = f == 0.f ? 0.f : f * x[n][half * 2], v1 = f == 0.f ? 0.f : f * x[n][half * 2 + 1];
        krow[half] = __fmaf_rn(__low2float(k), v0, __fmaf_rn(__high2float(k), v1, krow[half]));
        dk[n][half * 2] = __fmaf_rn(b, v0, dk[n][half * 2]);
        dk[n][half * 2 + 1] = __fmaf_rn(b, v1, dk[n][half * 2 + 1]);
      }
    }
    product<false, kLd, 0, false, kLd, kRows, 4>(oy, o, sh.y[0], m0, n0);
    product<false, kLd, kRows, false, kLd, kRows, 4>(ry, r, sh.y[0], m0, n0);
    __syncthreads();
    if (t + 1 < steps) load_b(t + 1);
    if ((t + 1) % slices) continue;
    // K K^T and Q K^T where this warp has dR Y^T and dO Y^T
    float kk[2][4], qk[2][4];
    zero(kk);
    zero(qk);
    product<false, LD, 0, false, LD, 0, DK / 16>(kk, sh.k, sh.k, m0, n0);
    product<false, LD, 0, false, LD, 0, DK / 16>(qk, sh.q, sh.k, m0, n0);
#pragma unroll
    for (int n = 0; n < 2; n++) {
      float col[2] = {0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8, j = n0 + n * 8 + (lane & 3) * 2;
        float po[2], mm[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int e = half * 2 + c;
          const bool low = j + c <= i, strict = j + c < i;
          const float f = low ? decay(sh.d, i, j + c) : 0.f, b = sh.d.beta[j + c];
          const float ov = low ? a.scale * f * oy[n][e] : 0.f, rv = strict ? f * ry[n][e] : 0.f;
          po[c] = b * ov;
          mm[c] = -b * rv;
          qrow[half] += (low ? qk[n][e] * po[c] : 0.f) + (strict ? kk[n][e] * mm[c] : 0.f);
          col[c] += (low ? qk[n][e] * ov : 0.f) - (strict ? kk[n][e] * rv : 0.f);
        }
        put2<kLd>(sh.p[0], sh.p[1], i, j, po[0], po[1]);
        put2<kLd>(sh.m[0], sh.m[1], i, j, mm[0], mm[1]);
      }
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int w = 4; w < 32; w *= 2) col[c] += __shfl_xor_sync(0xffffffffu, col[c], w);
      if (lane < 4) {
        sh.col[wr][n0 + n * 8 + lane * 2] = col[0];
        sh.col[wr][n0 + n * 8 + lane * 2 + 1] = col[1];
      }
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
#pragma unroll
      for (int w = 1; w < 4; w *= 2) {
        qrow[half] += __shfl_xor_sync(0xffffffffu, qrow[half], w);
        krow[half] += __shfl_xor_sync(0xffffffffu, krow[half], w);
      }
      if ((lane & 3) == 0) {
        sh.row[wc][i0 + half * 8] = qrow[half];
        sh.krow[wc][i0 + half * 8] = krow[half];
      }
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, w);
    if (lane == 0) sh.sum[warp] = inner;
    __syncthreads();
    product_part<false, kLd, kRows, true, LD, 0>(dq, sh.p[0], sh.k, m0, d0, 0, wr + 1);
    product_part<true, kLd, kRows, true, LD, 0>(dk, sh.p[0], sh.q, m0, d0, wr, 4);
    product_part<false, kLd, kRows, true, LD, 0>(dk, sh.m[0], sh.k, m0, d0, 0, wr + 1);
    product_part<true, kLd, kRows, true, LD, 0>(dk, sh.m[0], sh.k, m0, d0, wr, 4);
    if (warp == 0) {  // dbeta, and dg by sums of W's rows less its columns from the chunk's end, cut at resets
      const float keep = sh.d.since[kC - 1];
      float end = 0.f, sum[2];
      int era[2];
#pragma unroll
      for (int w = 0; w < 16; w++) end += sh.sum[w];
      end = keep == 0.f ? 0.f : keep * end;
      float tail = 0.f;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = half * 32 + lane;
        const float kd = (sh.krow[0][i] + sh.krow[1][i]) + (sh.krow[2][i] + sh.krow[3][i]);
        const float c = (sh.col[0][i] + sh.col[1][i]) + (sh.col[2][i] + sh.col[3][i]);
        if (i < len) p.dbeta[(start + i) * a.hv + h] = kd + c;
        tail += sh.d.beta[i] * kd;  // F_i u_i . (K_i dS')
        sum[half] = (sh.row[0][i] + sh.row[1][i]) + (sh.row[2][i] + sh.row[3][i]) - sh.d.beta[i] * (kd + c);
        era[half] = sh.d.era[i];
      }
#pragma unroll
      for (int w = 16; w; w >>= 1) tail += __shfl_xor_sync(0xffffffffu, tail, w);
      const int last = __shfl_sync(0xffffffffu, era[1], 31);
      float behind = end + tail;  // of the tokens behind this half, as far as they are of era `last`
      int behind_era = last;
#pragma unroll
      for (int half = 1; half >= 0; half--) {
        float v = sum[half];
#pragma unroll
        for (int w = 1; w < 32; w *= 2) {
          const float up = __shfl_down_sync(0xffffffffu, v, w);
          const int ue = __shfl_down_sync(0xffffffffu, era[half], w);
          if (lane + w < 32 && ue == era[half]) v += up;
        }
        if (era[half] == behind_era) v += behind;
        const int i = half * 32 + lane;
        const bool reset = i < len && a.g[(start + i) * a.hv + h] < -104.f;
        if (i < len) p.dg[(start + i) * a.hv + h] = reset ? 0.f : v;
        behind = __shfl_sync(0xffffffffu, v, 0);
        behind_era = __shfl_sync(0xffffffffu, era[half], 0);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int i = i0 + half * 8;
    if (i >= len) continue;
    const long to = ((start + i) * a.hk + kh) * a.dk;
#pragma unroll
    for (int n = 0; n < NK; n++) {
      const int j = d0 + n * 8 + (lane & 3) * 2;
      if (a.dk % 2 == 0 && j + 1 < a.dk) {
        *reinterpret_cast<__nv_bfloat162*>(p.dq + to + j) = __floats2bfloat162_rn(dq[n][half * 2], dq[n][half * 2 + 1]);
        *reinterpret_cast<__nv_bfloat162*>(p.dk + to + j) = __floats2bfloat162_rn(dk[n][half * 2], dk[n][half * 2 + 1]);
      } else {
#pragma unroll
        for (int c = 0; c < 2; c++)
          if (j + c < a.dk) {
            p.dq[to + j + c] = __float2bfloat16_rn(dq[n][half * 2 + c]);
            p.dk[to + j + c] = __float2bfloat16_rn(dk[n][half * 2 + c]);
          }
      }
    }
  }
}
// Rows that no sequence holds: their gradients are zero.
__global__ void __launch_bounds__(256) delta_rest_kernel(const GradArgs p) {
  grid_wait();
  grid_next();
  const DeltaArgs& a = p.d;
  long from, to, unused;
  seq_bounds(a, 0, from, unused);
  seq_bounds(a, a.seqs - 1, unused, to);
  for (long row = blockIdx.x; row < from + (a.n - to); row += gridDim.x) {
    const long r = row < from ? row : to + row - from;
    for (int i = threadIdx.x; i < a.hk * a.dk; i += 256)
      p.dq[r * a.hk * a.dk + i] = p.dk[r * a.hk * a.dk + i] = __float2bfloat16_rn(0.f);
    for (int i = threadIdx.x; i < a.hv; i += 256) p.dg[r * a.hv + i] = p.dbeta[r * a.hv + i] = 0.f;
  }
}

// ---------------------------------------------------------------------------------------------- host side
static int check_shape(const char* me, const pl_delta_shape* s, bool step) {
  PL_REQUIRE(s, PL_ERR_INVALID, "%s: NULL shape", me);
  PL_REQUIRE(s->dk >= 1 && s->dk <= 128, PL_ERR_INVALID, "%s: dk = %zu, 1 to 128 wanted", me, s->dk);
  PL_REQUIRE(s->dv >= 1 && s->dv <= 1024, PL_ERR_INVALID, "%s: dv = %zu, 1 to 1024 wanted", me, s->dv);
  PL_REQUIRE(s->heads_k >= 1 && s->heads_v >= s->heads_k && s->heads_v % s->heads_k == 0 && s->heads_v <= 4096,
             PL_ERR_INVALID, "%s: %zu heads of values for %zu of keys: a multiple of them, up to 4096, wanted", me, s->heads_v,
             s->heads_k);
  PL_REQUIRE(s->tokens <= (1u << 30) / s->heads_v, PL_ERR_INVALID, "%s: %zu tokens of %zu heads are too many", me, s->tokens,
             s->heads_v);
  PL_REQUIRE(step || s->sequences <= 65535, PL_ERR_INVALID, "%s: %zu sequences, at most 65535 wanted", me, s->sequences);
  PL_REQUIRE(s->scale == s->scale, PL_ERR_INVALID, "%s: scale = %g", me, s->scale);
  return PL_OK;
}
static bool rows16(const void* p, size_t ld, size_t hs) {
  return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && hs % 8 == 0;
}
static DeltaArgs delta_args(const pl_delta_shape* s, const void* q, const void* k, const void* v, const float* g,
                            const float* beta, const int32_t* offsets) {
  DeltaArgs a;
  a.n = (long)s->tokens;
  a.seqs = (int)s->sequences;
  a.hk = (int)s->heads_k;
  a.hv = (int)s->heads_v;
  a.dk = (int)s->dk;
  a.dv = (int)s->dv;
  a.dvp = (int)round_up((long)s->dv, 64);
  a.offsets = offsets;
  a.ldq = (long)s->q_token;
  a.hsq = (long)s->q_head;
  a.ldk = (long)s->k_token;
  a.hsk = (long)s->k_head;
  a.ldv = (long)s->v_token;
  a.hsv = (long)s->v_head;
  a.q = (const __nv_bfloat16*)q;
  a.k = (const __nv_bfloat16*)k;
  a.v = (const __nv_bfloat16*)v;
  a.g = g;
  a.beta = beta;
  a.scale = (float)s->scale;
  a.vec = rows16(q, s->q_token, s->q_head) && rows16(k, s->k_token, s->k_head) && rows16(v, s->v_token, s->v_head);
  return a;
}
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static size_t heads_slots(const pl_delta_shape* s) {
  return (size_t)slot_count((long)s->tokens, (long)s->sequences) * s->heads_v;
}
static size_t mats_bytes(const pl_delta_shape* s) { return up256(heads_slots(s) * sizeof(Mats)); }
static size_t states_bytes(const pl_delta_shape* s) { return up256(heads_slots(s) * s->dk * round_up((long)s->dv, 64) * 4); }
static size_t rows_bytes(const pl_delta_shape* s) { return up256(heads_slots(s) * kC * round_up((long)s->dv, 64) * 4); }

template <typename A>
static int launch_wide(void (*kernel)(A), dim3 grid, int threads, size_t smem, cudaStream_t st, const A& args) {
  int rc = raise_smem((const void*)kernel, smem);
  if (rc) return rc;
  PL_CUDA(launch_early(kernel, grid, dim3(threads), smem, st, args));
  count_launch();
  return PL_OK;
}
static int prep(const DeltaArgs& a, Mats* mats, cudaStream_t st) {
  const dim3 grid((unsigned)slot_count(a.n, a.seqs), (unsigned)a.hk);
  const bool wide = a.dk > 64;
  const size_t smem = wide ? sizeof(PrepShared<128>) : sizeof(PrepShared<64>);
  auto kernel = wide ? delta_prep_kernel<128> : delta_prep_kernel<64>;
  int rc = raise_smem((const void*)kernel, smem);
  if (rc) return rc;
  PL_CUDA(launch_early(kernel, grid, dim3(kPrepThreads), smem, st, a, mats));
  count_launch();
  return PL_OK;
}
template <int VEC>
static int step_launch(const StepArgs& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.d.n * p.d.hv), (unsigned)ceil_div(p.d.dv, 32 * VEC));
  PL_CUDA(p.d.dk <= 64 ? launch_early(delta_step_kernel<VEC, 8>, grid, dim3(256), 0, st, p)
                       : launch_early(delta_step_kernel<VEC, 16>, grid, dim3(256), 0, st, p));
  count_launch();
  return PL_OK;
}

}  // namespace pl

extern "C" {

size_t pl_delta_saved(const pl_delta_shape* s) {
  if (!s || s->sequences == 0) return 0;
  return pl::states_bytes(s) + pl::rows_bytes(s);
}
size_t pl_delta_ws(const pl_delta_shape* s, uint8_t grad) {
  if (!s || s->sequences == 0) return 0;
  return pl::mats_bytes(s) + (grad ? pl::states_bytes(s) + pl::rows_bytes(s) : 0);
}

int pl_delta_dev(const pl_delta_shape* s, const void* q, const void* k, const void* v, const float* g, const float* beta,
                 const int32_t* offsets, const float* state, void* o, float* final_state, void* saved, size_t saved_bytes,
                 void* ws, size_t ws_bytes, void* stream) {
  using namespace pl;
  const char* me = "pl_delta_dev";
  int rc = check_shape(me, s, false);
  if (rc) return rc;
  PL_REQUIRE(s->sequences > 0 || s->tokens == 0, PL_ERR_INVALID, "%s: tokens of no sequence", me);
  PL_REQUIRE(offsets || s->sequences == 0 || s->tokens % s->sequences == 0, PL_ERR_INVALID,
             "%s: %zu tokens are not %zu sequences of one length", me, s->tokens, s->sequences);
  if (s->sequences == 0) return PL_OK;
  PL_REQUIRE(final_state && (s->tokens == 0 || (q && k && v && g && beta && o)), PL_ERR_INVALID,
             "%s: NULL inputs or results", me);
  PL_REQUIRE(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= pl_delta_ws(s, 0), PL_ERR_INVALID,
             "%s: %zu bytes of workspace at 256 bytes needed", me, pl_delta_ws(s, 0));
  PL_REQUIRE(!saved || ((uintptr_t)saved % 256 == 0 && saved_bytes >= pl_delta_saved(s)), PL_ERR_INVALID,
             "%s: %zu bytes at 256 bytes needed for the gradient's states", me, pl_delta_saved(s));
  rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const DeltaArgs a = delta_args(s, q, k, v, g, beta, offsets);
  if (s->tokens) {
    rc = prep(a, (Mats*)ws, st);
    if (rc) return rc;
  }
  ScanArgs p = {a, (const Mats*)ws, state, (__nv_bfloat16*)o, final_state, nullptr, nullptr};
  if (saved) {
    p.kept = (__nv_bfloat16*)saved;
    p.y = (__nv_bfloat16*)((char*)saved + states_bytes(s));
  }
  const dim3 grid((unsigned)(a.dvp / 64), (unsigned)a.hv, (unsigned)a.seqs);
  return a.dk > 64 ? launch_wide(delta_scan_kernel<128>, grid, kScanThreads, sizeof(ScanShared<128>), st, p)
                   : launch_wide(delta_scan_kernel<64>, grid, kScanThreads, sizeof(ScanShared<64>), st, p);
}

int pl_delta_grad_dev(const pl_delta_shape* s, const void* dout, size_t do_token, size_t do_head, const float* dfinal,
                      const void* q, const void* k, const void* v, const float* g, const float* beta,
                      const int32_t* offsets, const void* saved, size_t saved_bytes, void* dq, void* dk, void* dv, float* dg,
                      float* dbeta, float* dstate, void* ws, size_t ws_bytes, void* stream) {
  using namespace pl;
  const char* me = "pl_delta_grad_dev";
  int rc = check_shape(me, s, false);
  if (rc) return rc;
  PL_REQUIRE(s->sequences > 0 || s->tokens == 0, PL_ERR_INVALID, "%s: tokens of no sequence", me);
  PL_REQUIRE(offsets || s->sequences == 0 || s->tokens % s->sequences == 0, PL_ERR_INVALID,
             "%s: %zu tokens are not %zu sequences of one length", me, s->tokens, s->sequences);
  if (s->sequences == 0) return PL_OK;
  PL_REQUIRE(s->tokens == 0 || (dout && q && k && v && g && beta && dq && dk && dv && dg && dbeta), PL_ERR_INVALID,
             "%s: NULL inputs or results", me);
  PL_REQUIRE(saved && (uintptr_t)saved % 256 == 0 && saved_bytes >= pl_delta_saved(s), PL_ERR_INVALID,
             "%s: the forward call's states (%zu bytes at 256 bytes) are needed", me, pl_delta_saved(s));
  PL_REQUIRE(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= pl_delta_ws(s, 1), PL_ERR_INVALID,
             "%s: %zu bytes of workspace at 256 bytes needed", me, pl_delta_ws(s, 1));
  rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const DeltaArgs a = delta_args(s, q, k, v, g, beta, offsets);
  char* w = (char*)ws;
  __nv_bfloat16 *ds = (__nv_bfloat16*)(w + mats_bytes(s)), *dr = (__nv_bfloat16*)(w + mats_bytes(s) + states_bytes(s));
  const bool vec_o = rows16(dout, do_token, do_head);
  if (s->tokens) {
    rc = prep(a, (Mats*)ws, st);
    if (rc) return rc;
  }
  const BackArgs b = {a, (const Mats*)ws, (const __nv_bfloat16*)dout, (long)do_token, (long)do_head, vec_o, dfinal,
                      (__nv_bfloat16*)dv, dstate, ds, dr};
  const dim3 grid((unsigned)(a.dvp / 64), (unsigned)a.hv, (unsigned)a.seqs);
  rc = a.dk > 64 ? launch_wide(delta_back_kernel<128>, grid, kScanThreads, sizeof(BackShared<128>), st, b)
                 : launch_wide(delta_back_kernel<64>, grid, kScanThreads, sizeof(BackShared<64>), st, b);
  if (rc || s->tokens == 0) return rc;
  const GradArgs p = {a, (const __nv_bfloat16*)dout, (long)do_token, (long)do_head, vec_o, (const __nv_bfloat16*)saved,
                      (const __nv_bfloat16*)((const char*)saved + states_bytes(s)), ds, dr, (__nv_bfloat16*)dq, (__nv_bfloat16*)dk,
                      dg, dbeta};
  const dim3 chunks((unsigned)slot_count(a.n, a.seqs), (unsigned)a.hk);
  rc = a.dk > 64 ? launch_wide(delta_grad_kernel<128>, chunks, kScanThreads, sizeof(GradShared<128>), st, p)
                 : launch_wide(delta_grad_kernel<64>, chunks, kScanThreads, sizeof(GradShared<64>), st, p);
  if (rc || !offsets) return rc;
  PL_CUDA(launch_early(delta_rest_kernel, dim3(64), dim3(256), 0, st, p));
  count_launch();
  return PL_OK;
}

int pl_delta_step_dev(const pl_delta_shape* s, const void* q, const void* k, const void* v, const float* g,
                      const float* beta, const float* state, float* state_out, void* o, void* stream) {
  using namespace pl;
  const char* me = "pl_delta_step_dev";
  int rc = check_shape(me, s, true);
  if (rc) return rc;
  if (s->tokens == 0) return PL_OK;
  PL_REQUIRE(q && k && v && g && beta && state && state_out && o, PL_ERR_INVALID, "%s: NULL inputs or results", me);
  rc = require_device();
  if (rc) return rc;
  const StepArgs p = {delta_args(s, q, k, v, g, beta, nullptr), state, state_out, (__nv_bfloat16*)o};
  const uintptr_t both = (uintptr_t)state | (uintptr_t)state_out;
  cudaStream_t st = (cudaStream_t)stream;
  if (s->dv % 4 == 0 && both % 16 == 0 && s->dv > 64) return step_launch<4>(p, st);
  if (s->dv % 2 == 0 && both % 8 == 0 && s->dv > 32) return step_launch<2>(p, st);
  return step_launch<1>(p, st);
}

}  // extern "C"
