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
//   dbeta_t = Z_t . Y_t with dR = diag(beta) Z
//   dg_t = sum over i >= t of (o_i . dO_i - v_i . dR_i), and <S', dS'> = exp(G_last) <S, dS'> + sum_j U_j . (F K dS')_j
//
// (dg up to the next reset: behind one, neither tokens nor S' depend on g_t).
//
// X and P depend on q, k, g and beta alone: one kernel makes them for all chunks at once. What is left in the chain over a
// sequence's chunks is a few products with the state, for each 64 columns of v on their own (columns do not mix), and
// what dq and dk need beyond the two chains (S per chunk forward, dS' back) is again one kernel over all chunks.
// What f32 results come from is held in f32: states, Y, Z and the outputs between the kernels, and as operands of products
// as three bf16 parts, which hold all 24 bits; f32 results are 1e-7 to 5e-7 off 64 bits, as with f32 operations. dq, dk and, without
// a gradient, o are bf16 and nothing else: two parts, 3e-6 (the rounding: 1.7e-3; with one part they would be 2e-3 off).
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
  using Word = typename std::conditional<VEC == 4, float4, typename std::conditional<VEC == 2, float2, float>::type>::type;
  // read and written once: past the caches (256 rows x 16 heads of 128 x 128: 105 -> 96 us)
  __device__ __forceinline__ void load(const float* p) {
    const Word w = __ldcs(reinterpret_cast<const Word*>(p));
    memcpy(v, &w, sizeof(w));
  }
  __device__ __forceinline__ void store(float* p) const {
    Word w;
    memcpy(&w, v, sizeof(w));
    __stcs(reinterpret_cast<Word*>(p), w);
  }
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
      x[r].load(s + (long)i * a.dv + col);
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
    x[r].store(to + (long)i * a.dv + col);
  }
}

// ---------------------------------------------------------------------------------------------- X and P of all chunks
// Per slot and value head: X and P, triangular, as three bf16 parts each, and the decays; per slot and key head K and Q in
// rows as they stand in shared memory, [2][64][dkp + 8], so that the other kernels get them by one bulk copy; per slot its
// chunk's first token and length (0: none).
// Measured: 8,192 chunks of a head, dk = 128, in 218 us, where their 820 MB would take 125: a block's dozen steps (search,
// copies, decays, two products, the inverse in blocks of 16 and 32) wait for one another, four blocks to an SM.
struct __align__(16) Mats {
  __nv_bfloat16 x[3][kTri], p[3][kTri];
  Decay d;
};

template <int DK>
constexpr uint32_t kTileBytes = 2 * kC * (DK + 8) * 2;
template <int DK>
__device__ __forceinline__ long tile_at(const DeltaArgs& a, long slot, int kh) {
  return (slot * a.hk + kh) * 2 * kC * (DK + 8);
}

// beta where it divides: not zero. What it adds to X is 1e-12 of what is there.
__device__ __forceinline__ float beta_of(float b) { return fabsf(b) < 1e-12f ? copysignf(1e-12f, b) : b; }
constexpr int kPrepThreads = 128;
template <int DK>
struct PrepShared {
  union {
    struct {
      __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)];
    };
    struct {  // when K K^T and Q K^T are in registers
      float at[kC][kC + 4];  // N diag(beta), transposed: [j][i]; above its diagonal, nothing is read
      float x[kC][kC + 4];   // its inverse with I
      float y[32][36];
    };
  };
  Decay d;
};
// out = -B (A C) for square blocks of S rows: A = at (transposed) at (r, c), C = x at (c, c), B = x at (r, r), out = x at
// (r, c); N threads per block of the matrix, thread t of them; `y` for A C.
template <int S, int N, typename Shared>
__device__ __forceinline__ void inverse_block(Shared& sh, float (*y)[36], int r, int c, int t) {
  constexpr int E = S * S / N, P = S / E;  // values per thread, threads per row
  const int i = t / P, j0 = t % P * E;
  float s[E];
#pragma unroll
  for (int e = 0; e < E; e++) s[e] = 0.f;
#pragma unroll 8
  for (int k = 0; k < S; k++) {
    const float f = sh.at[c + k][r + i];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(&sh.x[c + k][c + j0 + e]);
      s[e] = __fmaf_rn(f, v.x, s[e]), s[e + 1] = __fmaf_rn(f, v.y, s[e + 1]);
      s[e + 2] = __fmaf_rn(f, v.z, s[e + 2]), s[e + 3] = __fmaf_rn(f, v.w, s[e + 3]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(&y[i][j0 + e]) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) s[e] = 0.f;
#pragma unroll 8
  for (int k = 0; k < S; k++) {
    const float f = -sh.x[r + i][r + k];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(&y[k][j0 + e]);
      s[e] = __fmaf_rn(f, v.x, s[e]), s[e + 1] = __fmaf_rn(f, v.y, s[e + 1]);
      s[e + 2] = __fmaf_rn(f, v.z, s[e + 2]), s[e + 3] = __fmaf_rn(f, v.w, s[e + 3]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; e += 4)
    *reinterpret_cast<float4*>(&sh.x[r + i][c + j0 + e]) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
  __syncthreads();
}
template <int DK>
__global__ void __launch_bounds__(kPrepThreads, 4) delta_prep_kernel(
    const DeltaArgs a, Mats* __restrict__ mats, __nv_bfloat16* __restrict__ tiles, int2* __restrict__ table) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  PrepShared<DK>& sh = *reinterpret_cast<PrepShared<DK>*>(mem);
  constexpr int LD = DK + 8;
  const long slot = blockIdx.x;
  const int kh = blockIdx.y, group = a.hv / a.hk, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long start;
  const int len = slot_chunk(a, slot, start);
  if (kh == 0 && tid == 0) table[slot] = make_int2((int)start, len);
  if (len == 0) return;
  const Gates gates = load_gates(a, start, len, kh * group);
  copy_tile<DK, LD, kPrepThreads>(sh.k, a.k + start * a.ldk + kh * a.hsk, a.ldk, len, a.dk, a.vk, tid);
  copy_tile<DK, LD, kPrepThreads>(sh.q, a.q + start * a.ldq + kh * a.hsq, a.ldq, len, a.dk, a.vq, tid);
  cp_commit();
  chunk_decay(sh.d, gates);
  cp_wait<0>();
  tc::fence_proxy_async_smem();
  __syncthreads();
  if (tid == 0) {
    bulk_out(tiles + tile_at<DK>(a, slot, kh), sh.k, kTileBytes<DK>);
    tc::bulk_commit();
  }
  float kk[8][4], qk[8][4];  // rows 16 warp.. of K K^T and Q K^T, up to the diagonal's block
  zero(kk);
  zero(qk);
  {
    const uint32_t pk = smem_u32(sh.k + warp * 16 * LD + lane_a<false, LD>()), pq = pk + kC * LD * 2;
    const uint32_t pb = smem_u32(sh.k + lane_b<false, LD>());
#pragma unroll
    for (int k = 0; k < DK / 16; k++) {
      uint32_t x[4], y[4];
      ldsm<false>(x, pk + k * 32);
      ldsm<false>(y, pq + k * 32);
#pragma unroll
      for (int n = 0; n < 4; n++) {
        if (n > warp) continue;
        uint32_t b[4];
        ldsm<false>(b, pb + n * 32 * LD + k * 32);
        mma(kk[2 * n], x, b[0], b[1]);
        mma(kk[2 * n + 1], x, b[2], b[3]);
        mma(qk[2 * n], y, b[0], b[1]);
        mma(qk[2 * n + 1], y, b[2], b[3]);
      }
    }
  }
  if (tid == 0) tc::bulk_wait_read<0>();  // the places of K and Q are used again
  for (int e = 0; e < group; e++) {
    const int h = kh * group + e;
    Mats& out = mats[slot * a.hv + h];
    __syncthreads();
    if (e) {
      chunk_decay(sh.d, load_gates(a, start, len, h));
      __syncthreads();
    }
    if (tid < (int)(sizeof(Decay) / 16)) reinterpret_cast<uint4*>(&out.d)[tid] = reinterpret_cast<const uint4*>(&sh.d)[tid];
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int i = warp * 16 + half * 8 + (lane >> 2), ei = sh.d.era[i];
      const float2 ci = sh.d.cum[i];
#pragma unroll
      for (int t = 0; t < 8; t++) {
        if (t / 2 > warp) continue;
        const int j = t * 8 + (lane & 3) * 2;
        float p[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const float f = j + c <= i ? decay(ci, ei, sh.d, j + c) : 0.f;
          p[c] = j + c <= i ? qk[t][half * 2 + c] * f : 0.f;
          sh.at[j + c][i] = j + c < i ? kk[t][half * 2 + c] * f * beta_of(sh.d.beta[j + c]) : 0.f;
        }
        Parts<3> s;
        split<3>(p[0], p[1], s, 0);
#pragma unroll
        for (int c = 0; c < 3; c++) *reinterpret_cast<uint32_t*>(out.p[c] + tri_at(i, j)) = s.p[c][0];
      }
    }
    __syncthreads();
    // the inverse's four diagonal blocks of 16, a column per thread: x_i -= A_ij x_j as soon as x_j is known
    if (tid < 64) {
      const int b = tid & 48, c = tid & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < 15; j++)
#pragma unroll
        for (int i = (j + 1) & 12; i < 16; i += 4) {  // (up to the diagonal a row of `at` is zero)
          const float4 f = *reinterpret_cast<const float4*>(&sh.at[b + j][b + i]);
          x[i] = __fmaf_rn(-f.x, x[j], x[i]);
          x[i + 1] = __fmaf_rn(-f.y, x[j], x[i + 1]);
          x[i + 2] = __fmaf_rn(-f.z, x[j], x[i + 2]);
          x[i + 3] = __fmaf_rn(-f.w, x[j], x[i + 3]);
        }
#pragma unroll
      for (int i = 0; i < 16; i++) sh.x[b + i][b + c] = x[i];
    }
    __syncthreads();
    inverse_block<16, 64>(sh, sh.y + (tid >> 6) * 16, (tid >> 6) * 32 + 16, (tid >> 6) * 32, tid & 63);
    if (tid < 64) {  // above the diagonal blocks of 16 the blocks of 32 are zero
      const int b = tid & 32, r = tid & 31;
      if (r < 16)
#pragma unroll
        for (int c = 16; c < 32; c += 4) *reinterpret_cast<float4*>(&sh.x[b + r][b + c]) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    // the block below: -X22 (A21 X11), 4 x 4 values per thread, both first operands read along their rows: A21 lies transposed,
    // and X22 is put so where `at` is not used
    for (int i = tid; i < 32 * 32; i += kPrepThreads) sh.at[32 + (i & 31)][i >> 5] = sh.x[32 + (i >> 5)][32 + (i & 31)];
    __syncthreads();
    auto block_product = [&](const float (*m)[kC + 4], int m0, const float* c, int ldc, float sign, float (&s)[4][4]) {
      const int i0 = m0 + (tid >> 3) * 4, j0 = (tid & 7) * 4;
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll 8
      for (int k = 0; k < 32; k++) {
        const float4 u = *reinterpret_cast<const float4*>(&m[k][i0]), v = *reinterpret_cast<const float4*>(c + k * ldc + j0);
        const float ui[4] = {sign * u.x, sign * u.y, sign * u.z, sign * u.w}, vj[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) s[i][j] = __fmaf_rn(ui[i], vj[j], s[i][j]);
      }
    };
    if (tid < 64) {
      float s[4][4];
      block_product(sh.at, 32, sh.x[0], kC + 4, 1.f, s);
#pragma unroll
      for (int i = 0; i < 4; i++)
        *reinterpret_cast<float4*>(&sh.y[(tid >> 3) * 4 + i][(tid & 7) * 4]) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
    __syncthreads();
    if (tid < 64) {
      float s[4][4];
      block_product(sh.at + 32, 0, sh.y[0], 36, -1.f, s);
#pragma unroll
      for (int i = 0; i < 4; i++)
        *reinterpret_cast<float4*>(&sh.x[32 + (tid >> 3) * 4 + i][(tid & 7) * 4]) =
            make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    }
    __syncthreads();
#pragma unroll 5
    for (int i = tid; i < kTri / 2; i += kPrepThreads) {  // pair i of the ten blocks, in the order of rows and columns
      const int b = i >> 7, r = b < 1 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, c = b - r * (r + 1) / 2;
      const int y = r * 16 + (i >> 3 & 15), x = c * 16 + (i & 7) * 2;
      Parts<3> s;
      split<3>(sh.x[y][x], sh.x[y][x + 1], s, 0);
#pragma unroll
      for (int e = 0; e < 3; e++) *reinterpret_cast<uint32_t*>(out.x[e] + tri_at(y, x)) = s.p[e][0];
    }
  }
  if (tid == 0) tc::bulk_wait<0>();
}

// ---------------------------------------------------------------------------------------------- the chain forward
// What the chains leave for other kernels, f32, per slot, value head and 64 columns of v, as a warp's lanes hold it, four warps of 16
// columns one behind the other: states, and rows of 64 tokens.
__device__ __forceinline__ uint4* states_at(const DeltaArgs& a, const void* base, long slot, int h, int slice, int warp) {
  return (uint4*)base + (((slot * a.hv + h) * (a.dvp / 64) + slice) * 4 + warp) * (a.dkp / 8 * 32);
}
__device__ __forceinline__ uint4* lanes_at(const DeltaArgs& a, const void* base, long slot, int h, int slice, int warp) {
  return (uint4*)base + (((slot * a.hv + h) * (a.dvp / 64) + slice) * 4 + warp) * (8 * 32);
}

struct ScanArgs {
  DeltaArgs d;
  const Mats* mats;
  const __nv_bfloat16* tiles;
  const float* state;  // [seqs][hv][dk][dv], or NULL: zero
  __nv_bfloat16* o;    // [n][hv][dv]
  float* final_state;
  float *kept, *y, *out;  // for the gradient: S, Y and the f32 outputs of every slot
};
// A chunk's inputs, loaded while the chunk before it is worked on; x: 64 columns of v (forward), of dO (back).
template <int DK>
struct ChainIn {
  __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)], x[kC * kLd];
  Mats m;
};
// Four warps for the chain, 16 columns of v each, four for products beside it, four for memory.
constexpr int kChainThreads = 384;
constexpr int kAll = 15, kMovers = 14;  // barriers of all threads, of the four warps for memory
template <int DK>
struct ScanShared {
  ChainIn<DK> in[2];
  uint4 s[4][DK / 8 * 32];  // a warp's state, as its lanes hold it
  uint4 y[4][8 * 32];       // its Y
  uint64_t full[2];         // the inputs have come
};

// Rows that no sequence holds, in front of the first and behind the last: zero. Called by the blocks of those two.
template <int THREADS, typename T>
__device__ __forceinline__ void zero_rows(const DeltaArgs& a, int seq, T* out, long ld, int cols, int tid) {
  long from, to;
  seq_bounds(a, seq, from, to);
  for (int side = 0; side < 2; side++) {
    if (side ? seq != a.seqs - 1 : seq != 0) continue;
    const long r0 = side ? to : 0, r1 = side ? a.n : from;
    for (long i = r0 * cols + tid; i < r1 * cols; i += THREADS) out[i / cols * ld + i % cols] = T(0.f);
  }
}

// The state's columns of a warp, transposed, between memory [dk][dv] and registers [16 of dv][dk].
template <int NT>
__device__ __forceinline__ void state_in(float (&s)[NT][4], const float* src, int dk, int dv, int cols) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int j = (lane >> 2) + (e >> 1) * 8, i = t * 8 + (lane & 3) * 2 + (e & 1);
      s[t][e] = src && i < dk && j < cols ? src[(long)i * dv + j] : 0.f;
    }
}
template <int NT>
__device__ __forceinline__ void state_out(const float (&s)[NT][4], float* dst, int dk, int dv, int cols) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int j = (lane >> 2) + (e >> 1) * 8, i = t * 8 + (lane & 3) * 2 + (e & 1);
      if (i < dk && j < cols) dst[(long)i * dv + j] = s[t][e];
    }
}
// A warp's tiles from shared memory to memory, by its first lane; they may be written again when it returns.
__device__ __forceinline__ void lanes_out(void* dst, const void* src, uint32_t bytes) {
  if ((threadIdx.x & 31) == 0) {
    bulk_out(dst, src, bytes);
    tc::bulk_commit();
    tc::bulk_wait_read<0>();
  }
  __syncwarp();
}
// 64 rows of 16 values that this warp put at `tile`, to rows of `stride` in memory, `cols` of them.
__device__ __forceinline__ void rows_out(const __nv_bfloat16* tile, __nv_bfloat16* dst, long stride, int len, int cols,
                                         bool vec) {
  const int lane = threadIdx.x & 31;
  if (vec && cols >= 16) {
    for (int i = lane; i < len * 2; i += 32)
      *reinterpret_cast<uint4*>(dst + (i >> 1) * stride + (i & 1) * 8) =
          *reinterpret_cast<const uint4*>(tile + (i >> 1) * kLd + (i & 1) * 8);
  } else {
    for (int i = lane; i < len * 16; i += 32)
      if ((i & 15) < cols) dst[(i >> 4) * stride + (i & 15)] = tile[(i >> 4) * kLd + (i & 15)];
  }
}
// Where this lane's row of n-tiles 2 n, 2 n + 1 of an accumulator [16 of dv][tokens] goes in a tile of tokens.
__device__ __forceinline__ uint32_t across_at(const __nv_bfloat16* tile, int n) {
  const int lane = threadIdx.x & 31;
  return smem_u32(tile + (n * 16 + (lane & 7) + ((lane >> 4) & 1) * 8) * kLd + ((lane >> 3) & 1) * 8);
}

// A block per sequence, value head and 64 columns of v. A warp of the chain has 16 columns of the state, transposed [16][dk], and
// everything that a chunk makes of it: an accumulator's layout is that of a first operand, so K S, R, Y and F U go from one product
// into the next as they are, split into bf16 parts. The state is in shared memory, f32, as its lanes hold it (in registers, beside
// sums of parts of their own, 390 bytes spilled: 880 us instead of 704); the sums of a chunk are added to it in f32. What
// the next chunk's state does not wait for is another warp's, which reads the state and Y there: Q S and P U; a third one's is
// what goes from and to memory.
// A chunk takes 5.3 us, 9,900 clocks. Its products are 504 and, with or without a gradient, 312 or 188 of 16 x 8 x 16 for each
// scheduler, 8 clocks each: 6,528 or 5,536. Without K S it would be 1.2 us less, without F U K 0.9, without X R 0.5. (With two parts
// of each operand, 316 and 188 products, 3.9 us, and f32 results 3e-6 off.) 4 x 8,192 tokens of 16 heads of 128 x 128: 662 to
// 678 us, 128 of 148 SMs with a chain of 128 chunks each.
template <int DK, bool SAVE>
__global__ void __launch_bounds__(kChainThreads, 1) delta_scan_kernel(const ScanArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  ScanShared<DK>& sh = *reinterpret_cast<ScanShared<DK>*>(mem);
  constexpr int LD = DK + 8, NK = DK / 8, P = SAVE ? 3 : 2;  // parts of the outputs' operands
  const DeltaArgs& a = p.d;
  const int slice = blockIdx.x, c0 = slice * 64, h = blockIdx.y, seq = blockIdx.z, kh = h / (a.hv / a.hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5 & 3;
  const bool chain = threadIdx.x < 128;
  const int w0 = c0 + warp * 16, mine = a.dv - w0 < 16 ? a.dv - w0 : 16;  // this warp's columns (none: <= 0)
  long from, to;
  seq_bounds(a, seq, from, to);
  const long slot0 = from / kC + seq, chunks = (to - from + kC - 1) / kC;
  const int s_read = 1 + warp, y_ready = 5 + warp, k_done = 9 + warp;
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh.full[0], 1);
    tc::mbar_init(&sh.full[1], 1);
    tc::fence_mbar_init();
  }
  __syncthreads();
  if (chain) {
    float s[NK][4];
    const long sbase = ((long)seq * a.hv + h) * a.dk * a.dv + w0;
    state_in(s, p.state ? p.state + sbase : nullptr, a.dk, a.dv, mine);
#pragma unroll
    for (int t = 0; t < NK; t++) give(sh.s[warp], t, s[t]);
    for (long c = 0; c < chunks; c++) {
      ChainIn<DK>& in = sh.in[c & 1];
      if constexpr (SAVE) tc::fence_proxy_async_smem();  // bulk copies take S and Y
      meet<kChainThreads>(kAll);
      tc::mbar_wait(&sh.full[c & 1], c >> 1 & 1, a.err, PL_ERR_MBAR_TIMEOUT);
      float r[8][4], low[8][4];  // (K S)^T: [16 of dv][64 tokens]
      zero(r);
      zero(low);
      const uint32_t pk = smem_u32(in.k + lane_b<false, LD>());
#pragma unroll
      for (int k = 0; k < DK / 16; k++) {
        float s0[4], s1[4];
        take(sh.s[warp], 2 * k, s0);
        take(sh.s[warp], 2 * k + 1, s1);
        step<false, 4>(r, low, parts_of<3>(s0, s1), pk + k * 32, 32 * LD);
      }
      meet_arrive<64>(k_done);
      join(r, low);
      const uint32_t px = smem_u32(in.x + warp * 16 + lane_a<true, kLd>());
#pragma unroll
      for (int n = 0; n < 4; n++) {  // R = V - E K S
        uint32_t v[4];
        ldsm<true>(v, px + n * 32 * kLd);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const float2 f = *reinterpret_cast<const float2*>(in.m.d.since + n * 16 + t * 8 + (lane & 3) * 2);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float fe = e & 1 ? f.y : f.x;
            const uint32_t vv = v[t * 2 + (e >> 1)];
            float(&rr)[4] = r[2 * n + t];
            rr[e] = __uint_as_float(e & 1 ? vv & 0xffff0000u : vv << 16) - (fe == 0.f ? 0.f : fe * rr[e]);
          }
        }
      }
      float y[8][4];  // Y^T = R^T X^T
      zero(y);
      Parts<3> z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) z[k] = parts_of<3>(r[2 * k], r[2 * k + 1]);
      tri_product<false, 3, 3>(y, z, tri_lane<false>(in.m.x[0]));
#pragma unroll
      for (int t = 0; t < 8; t++) give(sh.y[warp], t, y[t]);
      if constexpr (SAVE) tc::fence_proxy_async_smem();
      meet_arrive<96>(y_ready);
      const float keep = in.m.d.since[kC - 1];
#pragma unroll
      for (int k = 0; k < 4; k++) {  // S^T += (F U)^T K
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const float2 f = *reinterpret_cast<const float2*>(in.m.d.until + k * 16 + t * 8 + (lane & 3) * 2);
          const float2 b = *reinterpret_cast<const float2*>(in.m.d.beta + k * 16 + t * 8 + (lane & 3) * 2);
          float(&u)[4] = y[2 * k + t];
          u[0] *= f.x * b.x, u[2] *= f.x * b.x;
          u[1] *= f.y * b.y, u[3] *= f.y * b.y;
        }
        z[k] = parts_of<3>(y[2 * k], y[2 * k + 1]);
      }
      meet<96>(s_read);
      token_steps<LD, NK>(z, smem_u32(in.k + lane_b<true, LD>()), [&](int t, const float(&add)[4]) {
        float v[4];
        take(sh.s[warp], t, v);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = __fmaf_rn(keep, keep == 0.f ? 0.f : v[e], add[e]);
        give(sh.s[warp], t, v);
      });
    }
    if (chunks) meet<kChainThreads>(kAll);
#pragma unroll
    for (int t = 0; t < NK; t++) take(sh.s[warp], t, s[t]);
    state_out(s, p.final_state + sbase, a.dk, a.dv, mine);
    return;
  }
  if (threadIdx.x < 256) {  // Q S, P U
    for (long c = 0; c < chunks; c++) {
      ChainIn<DK>& in = sh.in[c & 1];
      meet<kChainThreads>(kAll);
      tc::mbar_wait(&sh.full[c & 1], c >> 1 & 1, a.err, PL_ERR_MBAR_TIMEOUT);
      float o[8][4], low[8][4];  // (Q S)^T
      zero(o);
      zero(low);
      const uint32_t pq = smem_u32(in.q + lane_b<false, LD>());
      meet<64>(k_done);  // K S goes first: beside Q S it takes 0.3 us longer
#pragma unroll
      for (int k = 0; k < DK / 16; k++) {
        float s0[4], s1[4];
        take(sh.s[warp], 2 * k, s0);
        take(sh.s[warp], 2 * k + 1, s1);
        step<false, 4>(o, low, parts_of<P>(s0, s1), pq + k * 32, 32 * LD);
      }
      meet_arrive<96>(s_read);
      join(o, low);
#pragma unroll
      for (int t = 0; t < 8; t++) {
        const float2 f = *reinterpret_cast<const float2*>(in.m.d.since + t * 8 + (lane & 3) * 2);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float fe = e & 1 ? f.y : f.x;
          o[t][e] = fe == 0.f ? 0.f : fe * o[t][e];
        }
      }
      zero(low);
      meet<96>(y_ready);
      Parts<P> z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float u[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const float2 b = *reinterpret_cast<const float2*>(in.m.d.beta + k * 16 + t * 8 + (lane & 3) * 2);
          take(sh.y[warp], 2 * k + t, u[t]);
          u[t][0] *= b.x, u[t][2] *= b.x;
          u[t][1] *= b.y, u[t][3] *= b.y;
        }
        z[k] = parts_of<P>(u[0], u[1]);
      }
      tri_product<false, P, P>(low, z, tri_lane<false>(in.m.p[0]));
      join(o, low);
      // the chain has read these columns of v before it gave Y: o takes their place on its way out
#pragma unroll
      for (int n = 0; n < 4; n++) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[2 * n][e] *= a.scale, o[2 * n + 1][e] *= a.scale;
        store_across(across_at(in.x + warp * 16, n), o[2 * n], o[2 * n + 1]);
      }
      if constexpr (SAVE) {
        uint4* to = lanes_at(a, p.out, slot0 + c, h, slice, warp);
#pragma unroll
        for (int t = 0; t < 8; t++) give(to, t, o[t]);
      }
    }
    if (chunks) meet<kChainThreads>(kAll);
    return;
  }
  // memory
  const int tid = threadIdx.x - 256, cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
  auto load = [&](long c) {
    const long start = from + c * kC;
    const int len = (int)(to - start < kC ? to - start : kC);
    ChainIn<DK>& in = sh.in[c & 1];
    uint64_t* bar = &sh.full[c & 1];
    tc::fence_proxy_async_smem();  // what was there has been read the ordinary way
    if (tid == 0) {
      tc::mbar_expect_tx(bar, sizeof(Mats) + kTileBytes<DK>);
      bulk_in(in.k, p.tiles + tile_at<DK>(a, slot0 + c, kh), kTileBytes<DK>, bar);
      bulk_in(&in.m, p.mats + (slot0 + c) * a.hv + h, sizeof(Mats), bar);
    }
    copy_tile<64, kLd, 128>(in.x, a.v + start * a.ldv + h * a.hsv + c0, a.ldv, len, cols, a.vv, tid);
    cp_commit();
  };
  const bool vec_o = a.dv % 8 == 0 && (uintptr_t)p.o % 16 == 0;
  auto write_o = [&](long c) {
    const long start = from + c * kC;
    rows_out(sh.in[c & 1].x + warp * 16, p.o + start * a.hv * a.dv + (long)h * a.dv + w0, (long)a.hv * a.dv,
             (int)(to - start < kC ? to - start : kC), mine, vec_o);
  };
  if (chunks) load(0);
  zero_rows<128>(a, seq, p.o + (long)h * a.dv + c0, (long)a.hv * a.dv, cols, tid);
  for (long c = 0; c < chunks; c++) {
    cp_wait<0>();
    meet<kChainThreads>(kAll);
    if (c > 0) write_o(c - 1);
    meet<128>(kMovers);  // the place of chunk c - 1's inputs, and of its o, is free
    if (c + 1 < chunks) load(c + 1);
    if constexpr (SAVE) lanes_out(states_at(a, p.kept, slot0 + c, h, slice, warp), sh.s[warp], sizeof(sh.s[0]));
    meet_arrive<96>(s_read);
    meet<96>(y_ready);
    if constexpr (SAVE) lanes_out(lanes_at(a, p.y, slot0 + c, h, slice, warp), sh.y[warp], sizeof(sh.y[0]));
  }
  if (chunks) {
    meet<kChainThreads>(kAll);
    write_o(chunks - 1);
  }
  if constexpr (SAVE) tc::bulk_wait<0>();
}

// ---------------------------------------------------------------------------------------------- the chain back
struct BackArgs {
  DeltaArgs d;
  const Mats* mats;
  const __nv_bfloat16* tiles;
  const __nv_bfloat16* dout;  // [n][hv][dv], strides below
  long ldo, hso;
  int align_o;
  const float* dfinal;          // [seqs][hv][dk][dv], or NULL: zero
  const float *kept, *y, *out;  // of the forward pass: S, Y and the f32 outputs
  __nv_bfloat16* dv;            // [n][hv][dv]
  float* dstate;                // or NULL
  float *ds, *dr;               // dS' and dR of every slot
  float* sums;                  // sums_at
};
// Per slot, value head and 16 columns of v, sums over them: of every token Y . Z beta' and o . dO - v . dR; of the chunk <S', dS'> and
// <S, dS>, which is dg of its first token (zero, not nearly zero, without a state).
constexpr int kSums = 2 * kC + 2;
__device__ __forceinline__ long sums_at(const DeltaArgs& a, long slot, int h, int group) {
  return ((slot * a.hv + h) * (a.dvp / 16) + group) * kSums;
}
// A warp's sums over the 16 rows of an accumulator [16][64]; lane l gets those of columns 2 l and 2 l + 1.
__device__ __forceinline__ float2 column_sums(const float (&v)[8][2]) {
  const int lane = threadIdx.x & 31;
  float a[4][2], b[2][2], c[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
#pragma unroll
    for (int t = 0; t < 4; t++)
      a[t][e] = (lane & 16 ? v[t + 4][e] : v[t][e]) + __shfl_xor_sync(0xffffffffu, lane & 16 ? v[t][e] : v[t + 4][e], 16);
#pragma unroll
    for (int t = 0; t < 2; t++)
      b[t][e] = (lane & 8 ? a[t + 2][e] : a[t][e]) + __shfl_xor_sync(0xffffffffu, lane & 8 ? a[t][e] : a[t + 2][e], 8);
    c[e] = (lane & 4 ? b[1][e] : b[0][e]) + __shfl_xor_sync(0xffffffffu, lane & 4 ? b[0][e] : b[1][e], 4);
  }
  return make_float2(c[0], c[1]);
}
template <int DK>
struct BackShared {
  ChainIn<DK> in[2];
  __nv_bfloat16 v[kC * kLd];
  uint4 s[4][DK / 8 * 32];  // a warp's dS', as its lanes hold it
  uint4 x[4][8 * 32];       // scale P^T dO from the helper, then beta' Z to memory
  uint4 f[4][8 * 32];       // F K dS'
  uint64_t full[2];
};
// As the chain forward, from the last chunk to the first. The helpers' products, of dO with P and Q, need nothing of the chain; they add
// theirs to dS' when the chain and memory have read it, the chain its own after that.
// Memory's warps also make the gates' gradients of what passes through them, in f32: dbeta is Z . Y, token by token (X^T beta dU is
// beta Z; where beta is zero, a tiny one stands in), and dg is sums of o . dO - v . dR. 64 x 512 tokens of 8 heads of 128 x 128: 465 us,
// where its 1.7 GB would take 260 (forward, with what the gradient needs written out: 392 to 402).
template <int DK>
__global__ void __launch_bounds__(kChainThreads, 1) delta_back_kernel(const BackArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  BackShared<DK>& sh = *reinterpret_cast<BackShared<DK>*>(mem);
  constexpr int LD = DK + 8, NK = DK / 8;
  const DeltaArgs& a = p.d;
  const int slice = blockIdx.x, c0 = slice * 64, h = blockIdx.y, seq = blockIdx.z, kh = h / (a.hv / a.hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5 & 3;
  const bool chain = threadIdx.x < 128;
  const int w0 = c0 + warp * 16, mine = a.dv - w0 < 16 ? a.dv - w0 : 16;
  long from, to;
  seq_bounds(a, seq, from, to);
  const long slot0 = from / kC + seq, chunks = (to - from + kC - 1) / kC;
  constexpr int EP = 3;  // parts of E dR
  const int u_ready = 1 + warp, q_ready = 5 + warp, r_ready = 9 + warp;
  constexpr int kRead = 13;  // the chain and memory have read dS'
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh.full[0], 1);
    tc::mbar_init(&sh.full[1], 1);
    tc::fence_mbar_init();
  }
  __syncthreads();
  if (chain) {
    float s[NK][4];  // dS'^T
    const long sbase = ((long)seq * a.hv + h) * a.dk * a.dv + w0;
    state_in(s, p.dfinal ? p.dfinal + sbase : nullptr, a.dk, a.dv, mine);
#pragma unroll
    for (int t = 0; t < NK; t++) give(sh.s[warp], t, s[t]);
    for (long c = chunks - 1, it = 0; c >= 0; c--, it++) {
      ChainIn<DK>& in = sh.in[it & 1];
      tc::fence_proxy_async_smem();  // bulk copies take dS' and dR
      meet<kChainThreads>(kAll);
      tc::mbar_wait(&sh.full[it & 1], it >> 1 & 1, a.err, PL_ERR_MBAR_TIMEOUT);
      float x[8][4], low[8][4];  // (K dS')^T: [16 of dv][64 tokens]
      zero(x);
      zero(low);
      const uint32_t pk = smem_u32(in.k + lane_b<false, LD>());
#pragma unroll
      for (int k = 0; k < DK / 16; k++) {
        float s0[4], s1[4];
        take(sh.s[warp], 2 * k, s0);
        take(sh.s[warp], 2 * k + 1, s1);
        step<false, 4>(x, low, parts_of<3>(s0, s1), pk + k * 32, 32 * LD);
      }
      meet_arrive<kChainThreads>(kRead);
      join(x, low);
      meet<64>(u_ready);
#pragma unroll
      for (int t = 0; t < 8; t++) {  // beta' dU = beta' (F K dS' + scale P^T dO)
        const float2 b = *reinterpret_cast<const float2*>(in.m.d.beta + t * 8 + (lane & 3) * 2);
        const float2 f = *reinterpret_cast<const float2*>(in.m.d.until + t * 8 + (lane & 3) * 2);
        float u[4];
        take(sh.x[warp], t, u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float fe = e & 1 ? f.y : f.x;
          x[t][e] = fe == 0.f ? 0.f : fe * x[t][e];
        }
        give(sh.f[warp], t, x[t]);
#pragma unroll
        for (int e = 0; e < 4; e++) x[t][e] = beta_of(e & 1 ? b.y : b.x) * (x[t][e] + u[e]);
      }
      float r[8][4];  // (beta' Z)^T = (beta' dU)^T X
      zero(r);
      {
        Parts<3> z[4];
#pragma unroll
        for (int k = 0; k < 4; k++) z[k] = parts_of<3>(x[2 * k], x[2 * k + 1]);
        tri_product<true, 3, 3>(r, z, tri_lane<true>(in.m.x[0]));
      }
#pragma unroll
      for (int t = 0; t < 8; t++) give(sh.x[warp], t, r[t]);
      tc::fence_proxy_async_smem();
      meet_arrive<64>(r_ready);
      Parts<EP> z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {  // dS^T -= (E dR)^T K
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const float2 f = *reinterpret_cast<const float2*>(in.m.d.since + k * 16 + t * 8 + (lane & 3) * 2);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float fe = e & 1 ? f.y : f.x;
            r[2 * k + t][e] = fe == 0.f ? 0.f : -fe * r[2 * k + t][e];
          }
        }
        z[k] = parts_of<EP>(r[2 * k], r[2 * k + 1]);
      }
      meet<64>(q_ready);
      token_steps<LD, NK>(z, smem_u32(in.k + lane_b<true, LD>()), [&](int t, const float(&add)[4]) {
        float v[4];
        take(sh.s[warp], t, v);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += add[e];
        give(sh.s[warp], t, v);
      });
    }
    if (chunks) meet<kChainThreads>(kAll);
#pragma unroll
    for (int t = 0; t < NK; t++) take(sh.s[warp], t, s[t]);
    if (p.dstate) state_out(s, p.dstate + sbase, a.dk, a.dv, mine);
    return;
  }
  if (threadIdx.x < 256) {  // scale P^T dO and scale (E dO)^T Q
    for (long it = 0; it < chunks; it++) {
      ChainIn<DK>& in = sh.in[it & 1];
      meet<kChainThreads>(kAll);
      tc::mbar_wait(&sh.full[it & 1], it >> 1 & 1, a.err, PL_ERR_MBAR_TIMEOUT);
      const uint32_t px = smem_u32(in.x + warp * 16 + lane_a<true, kLd>());
      uint32_t o[4][4];  // dO^T: [16 of dv][64 tokens]
#pragma unroll
      for (int k = 0; k < 4; k++) ldsm<true>(o[k], px + k * 32 * kLd);
      {
        float u[8][4];
        zero(u);
        Parts<1> x[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) x[k].p[0][e] = o[k][e];
        tri_product<true, 1, 3>(u, x, tri_lane<true>(in.m.p[0]));
#pragma unroll
        for (int t = 0; t < 8; t++) {
#pragma unroll
          for (int e = 0; e < 4; e++) u[t][e] *= a.scale;
          give(sh.x[warp], t, u[t]);
        }
      }
      meet_arrive<64>(u_ready);
      Parts<3> z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float eo[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const float2 f = *reinterpret_cast<const float2*>(in.m.d.since + k * 16 + t * 8 + (lane & 3) * 2);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float fe = e & 1 ? f.y : f.x;
            const uint32_t oo = o[k][t * 2 + (e >> 1)];
            eo[t][e] = fe == 0.f ? 0.f : a.scale * fe * __uint_as_float(e & 1 ? oo & 0xffff0000u : oo << 16);
          }
        }
        z[k] = parts_of<3>(eo[0], eo[1]);
      }
      const float keep = in.m.d.since[kC - 1];
      meet<kChainThreads>(kRead);
      token_steps<LD, NK>(z, smem_u32(in.q + lane_b<true, LD>()), [&](int t, const float(&add)[4]) {
        float v[4];
        take(sh.s[warp], t, v);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = __fmaf_rn(keep, keep == 0.f ? 0.f : v[e], add[e]);
        give(sh.s[warp], t, v);
      });
      meet_arrive<64>(q_ready);
    }
    if (chunks) meet<kChainThreads>(kAll);
    return;
  }
  // memory
  const int tid = threadIdx.x - 256, cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
  auto load = [&](long c) {
    const long start = from + c * kC, it = chunks - 1 - c;
    const int len = (int)(to - start < kC ? to - start : kC);
    ChainIn<DK>& in = sh.in[it & 1];
    uint64_t* bar = &sh.full[it & 1];
    tc::fence_proxy_async_smem();
    if (tid == 0) {
      tc::mbar_expect_tx(bar, sizeof(Mats) + kTileBytes<DK>);
      bulk_in(in.k, p.tiles + tile_at<DK>(a, slot0 + c, kh), kTileBytes<DK>, bar);
      bulk_in(&in.m, p.mats + (slot0 + c) * a.hv + h, sizeof(Mats), bar);
    }
    copy_tile<64, kLd, 128>(in.x, p.dout + start * p.ldo + h * p.hso + c0, p.ldo, len, cols, p.align_o, tid);
  };
  if (chunks) load(chunks - 1);
  cp_commit();
  zero_rows<128>(a, seq, p.dv + (long)h * a.dv + c0, (long)a.hv * a.dv, cols, tid);
  float s[NK][4];  // S before a slot's chunk, and its product with the gradient in shared memory: this lane's part
  auto load_s = [&](long slot) {
    const uint4* from_s = states_at(a, p.kept, slot, h, slice, warp);
#pragma unroll
    for (int t = 0; t < NK; t++) take(from_s, t, s[t]);
  };
  auto inner = [&] {
    float f = 0.f;
#pragma unroll
    for (int t = 0; t < NK; t++) {
      float v[4];
      take(sh.s[warp], t, v);
#pragma unroll
      for (int e = 0; e < 4; e++) f = __fmaf_rn(s[t][e], v[e], f);
    }
    return f;
  };
  auto warp_total = [](float f) {
#pragma unroll
    for (int w = 16; w; w >>= 1) f += __shfl_xor_sync(0xffffffffu, f, w);
    return f;
  };
  const bool vec_dv = a.dv % 8 == 0 && (uintptr_t)p.dv % 16 == 0;
  for (long c = chunks - 1; c >= 0; c--) {
    const long start = from + c * kC, slot = slot0 + c;
    const int len = (int)(to - start < kC ? to - start : kC);
    ChainIn<DK>& in = sh.in[(chunks - 1 - c) & 1];
    cp_wait<0>();
    meet<kChainThreads>(kAll);
    copy_tile<64, kLd, 128>(sh.v, a.v + start * a.ldv + h * a.hsv + c0, a.ldv, len, cols, a.vv, tid);
    cp_commit();
    if (c > 0) load(c - 1);
    cp_commit();
    const uint4 *yf = lanes_at(a, p.y, slot, h, slice, warp), *of = lanes_at(a, p.out, slot, h, slice, warp);
    load_s(slot);
    lanes_out(states_at(a, p.ds, slot, h, slice, warp), sh.s[warp], sizeof(sh.s[0]));
    float fu = inner();
    meet_arrive<kChainThreads>(kRead);
    float y[8][4], o[8][4];
#pragma unroll
    for (int t = 0; t < 8; t++) {
      take(yf, t, y[t]);
      take(of, t, o[t]);
    }
    cp_wait<1>();
    meet<128>(kMovers);  // v is there
    tc::mbar_wait(&sh.full[(chunks - 1 - c) & 1], (chunks - 1 - c) >> 1 & 1, a.err, PL_ERR_MBAR_TIMEOUT);
    meet<64>(r_ready);
    const uint32_t px = smem_u32(in.x + warp * 16 + lane_a<true, kLd>()), pv = smem_u32(sh.v + warp * 16 + lane_a<true, kLd>());
    float zy[8][2], ov[8][2];
    const float keep = in.m.d.since[kC - 1];
    fu = keep == 0.f ? 0.f : keep * fu;  // and F K dS' . U: <S', dS'>
    lanes_out(lanes_at(a, p.dr, slot, h, slice, warp), sh.x[warp], sizeof(sh.x[0]));
#pragma unroll
    for (int n = 0; n < 4; n++) {
      uint32_t d4[4], v4[4];
      ldsm<true>(d4, px + n * 32 * kLd);
      ldsm<true>(v4, pv + n * 32 * kLd);
      float r[2][4];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const int tt = 2 * n + t;
        const float2 b = *reinterpret_cast<const float2*>(in.m.d.beta + tt * 8 + (lane & 3) * 2);
        float f[4];
        take(sh.x[warp], tt, r[t]);
        take(sh.f[warp], tt, f);
#pragma unroll
        for (int e = 0; e < 2; e++) zy[tt][e] = ov[tt][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t dd = d4[t * 2 + (e >> 1)], vv = v4[t * 2 + (e >> 1)];
          const float be = e & 1 ? b.y : b.x;
          zy[tt][e & 1] = __fmaf_rn(r[t][e], y[tt][e], zy[tt][e & 1]);
          if (be == 0.f) r[t][e] = 0.f;
          ov[tt][e & 1] = __fmaf_rn(o[tt][e], __uint_as_float(e & 1 ? dd & 0xffff0000u : dd << 16), ov[tt][e & 1]);
          ov[tt][e & 1] = __fmaf_rn(-r[t][e], __uint_as_float(e & 1 ? vv & 0xffff0000u : vv << 16), ov[tt][e & 1]);
          fu = __fmaf_rn(be * y[tt][e], f[e], fu);
        }
      }
      // this warp and the helper have read these columns of dO: dv takes their place on its way out
      store_across(across_at(in.x + warp * 16, n), r[0], r[1]);
    }
    float* sums = p.sums + sums_at(a, slot, h, slice * 4 + warp);
    reinterpret_cast<float2*>(sums)[lane] = column_sums(zy);
    reinterpret_cast<float2*>(sums + kC)[lane] = column_sums(ov);
    fu = warp_total(fu);
    if (lane == 0) {
      sums[2 * kC] = fu;
      if (c + 1 < chunks) p.sums[sums_at(a, slot + 1, h, slice * 4 + warp) + 2 * kC + 1] = fu;
    }
    __syncwarp();
    rows_out(in.x + warp * 16, p.dv + start * a.hv * a.dv + (long)h * a.dv + w0, (long)a.hv * a.dv, len, mine, vec_dv);
  }
  if (chunks) {
    load_s(slot0);
    meet<kChainThreads>(kAll);
    const float f = warp_total(inner());
    if (lane == 0) p.sums[sums_at(a, slot0, h, slice * 4 + warp) + 2 * kC + 1] = f;
  }
  tc::bulk_wait<0>();
}

// ---------------------------------------------------------------------------------------------- the other gradients
constexpr int kGradThreads = 512;
constexpr int kRows = kC * kLd;  // a 64 x 64 tile: the distance of its second part
struct GradArgs {
  DeltaArgs d;
  const __nv_bfloat16* dout;
  long ldo, hso;
  int align_o;
  const float *kept, *y, *ds, *dr, *sums;
  const Mats* mats;
  const __nv_bfloat16* tiles;
  const int2* table;
  __nv_bfloat16 *dq, *dk;  // [n][hk][dk]
  float *dg, *dbeta;       // [n][hv]
};
template <int DK>
struct GradShared {
  __nv_bfloat16 k[kC * (DK + 8)], q[kC * (DK + 8)];
  __nv_bfloat16 o[2][kC * kLd], r[2][2][kC * kLd];  // by turns: the next step's are on their way
  __nv_bfloat16 s[2][kC * (DK + 8)], ds[2][kC * (DK + 8)], y[2][kC * kLd];  // transposed, as r
  __nv_bfloat16 p[2][kC * kLd], m[2][kC * kLd];     // scale dO U^T * D, -M
  float gate[2 * kC + 2];
  Decay decay[2];  // by turns, a head's
  uint64_t full[2];  // S, dO, dR (and K, Q, the decays); dS', Y
};
// A tile [64 of dv][8 NT] in f32, as four warps' lanes hold it, that a block turns into two bf16 parts of it, [2][64][LD], at the same
// place: read by all, a barrier, written. (What it is needed for, dq and dk, is rounded to bf16. Written as parts by the chains, four
// bytes at a time, the three kernels took 1,480 us for 64 x 512 tokens of 8 heads; so they take 1,340.)
template <int NT>
struct F32Tile {
  static constexpr int N = NT * 128 / kGradThreads;
  uint4 v[N];
  __device__ __forceinline__ void take(const __nv_bfloat16* from, int tid) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = reinterpret_cast<const uint4*>(from)[i * kGradThreads + tid];
  }
  template <int LD>
  __device__ __forceinline__ void give(__nv_bfloat16* to, int tid) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int at = i * kGradThreads + tid, lane = at & 31, t = at / 32 % NT, w = at / 32 / NT;
      __nv_bfloat16* p = to + (w * 16 + (lane >> 2)) * LD + t * 8 + (lane & 3) * 2;
      put2<LD>(p, p + kC * LD, 0, 0, __uint_as_float(v[i].x), __uint_as_float(v[i].y));
      put2<LD>(p, p + kC * LD, 8, 0, __uint_as_float(v[i].z), __uint_as_float(v[i].w));
    }
  }
};
// A block per chunk and key head, 16 warps: its value heads one after the other, so that what they add to dq and dk stays in
// registers and is added in their order; of each, 64 columns of v after the other (a step). A step's loads are under
// way during the one before it. 4,096 chunks of a head in 474 us: 31,000 clocks each, of which the products take 15,000.
template <int DK>
__global__ void __launch_bounds__(kGradThreads) delta_grad_kernel(const GradArgs p) {
  grid_wait();
  grid_next();
  extern __shared__ __align__(16) unsigned char mem[];
  GradShared<DK>& sh = *reinterpret_cast<GradShared<DK>*>(mem);
  constexpr int LD = DK + 8, NK = DK / 32;  // n-tiles of a warp's quarter of dk
  constexpr int kState = kC * LD;           // the distance of a state's second part
  const DeltaArgs& a = p.d;
  const long slot = blockIdx.x;
  const int kh = blockIdx.y, group = a.hv / a.hk, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    tc::mbar_init(&sh.full[0], 1);
    tc::mbar_init(&sh.full[1], 1);
    tc::fence_mbar_init();
  }
  const int2 chunk = p.table[slot];
  const long start = chunk.x;
  if (start < 0 || start >= a.n || chunk.y <= 0) return;  // (inside the tensors, whatever `saved` holds)
  const int most = (int)(a.n - start < kC ? a.n - start : kC), len = chunk.y < most ? chunk.y : most;
  const int slices = a.dvp / 64, steps = group * slices;
  constexpr uint32_t kStateBytes = kC * DK * 4, kRowsBytes = kC * kC * 4;
  auto load_a = [&](int t) {  // S, dO, dR, a head's decays
    const int h = kh * group + t / slices, slice = t % slices, c0 = slice * 64;
    const int cols = a.dv - c0 < 64 ? a.dv - c0 : 64;
    if (tid == 64) {
      tc::mbar_expect_tx(&sh.full[0], kStateBytes + kRowsBytes + (slice == 0 ? sizeof(Decay) : 0) +
                                          (t == 0 ? kTileBytes<DK> : 0));
      if (t == 0) bulk_in(sh.k, p.tiles + tile_at<DK>(a, slot, kh), kTileBytes<DK>, &sh.full[0]);
      bulk_in(sh.s, states_at(a, p.kept, slot, h, slice, 0), kStateBytes, &sh.full[0]);
      bulk_in(sh.r[t & 1], lanes_at(a, p.dr, slot, h, slice, 0), kRowsBytes, &sh.full[0]);
      if (slice == 0) bulk_in(&sh.decay[t / slices & 1], &p.mats[slot * a.hv + h].d, sizeof(Decay), &sh.full[0]);
    }
    copy_tile<64, kLd, kGradThreads>(sh.o[t & 1], p.dout + start * p.ldo + h * p.hso + c0, p.ldo, len, cols, p.align_o, tid);
    cp_commit();
  };
  auto load_b = [&](int t) {  // dS', Y
    const int h = kh * group + t / slices, slice = t % slices;
    if (tid == 0) {
      tc::mbar_expect_tx(&sh.full[1], kStateBytes + kRowsBytes);
      bulk_in(sh.ds, states_at(a, p.ds, slot, h, slice, 0), kStateBytes, &sh.full[1]);
      bulk_in(sh.y, lanes_at(a, p.y, slot, h, slice, 0), kRowsBytes, &sh.full[1]);
    }
  };
  __syncthreads();
  load_a(0);
  load_b(0);
  const int wr = warp & 3, wc = warp >> 2, m0 = wr * 16, i0 = m0 + (lane >> 2);
  const int n0 = wc * 16, d0 = wc * (DK / 4);  // this warp's columns of a 64 x 64 tile, of a 64 x dk tile
  float dq[NK][4], dk[NK][4], oy[2][4], ry[2][4];
  zero(dq);
  zero(dk);
  for (int t = 0; t < steps; t++) {
    const int h = kh * group + t / slices;
    const __nv_bfloat16* o = sh.o[t & 1];
    const __nv_bfloat16* r = sh.r[t & 1][0];
    const Decay& d = sh.decay[t / slices & 1];
    if (t % slices == 0) {
      zero(oy);
      zero(ry);
      // the chain's sums of this head, by token; warp 4: of the chunk
      const float* sums = p.sums + sums_at(a, slot, h, 0);
      float v = 0.f;
      if (tid < 2 * kC) {
#pragma unroll 8
        for (int g = 0; g < a.dvp / 16; g++) v += sums[g * kSums + tid];
        sh.gate[tid] = v;
      } else if (warp == 4) {
        float u = 0.f;
        for (int g = lane; g < a.dvp / 16; g += 32) {
          v += sums[g * kSums + 2 * kC];
          u += sums[g * kSums + 2 * kC + 1];
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) {
          v += __shfl_xor_sync(0xffffffffu, v, w);
          u += __shfl_xor_sync(0xffffffffu, u, w);
        }
        if (lane == 0) {
          sh.gate[2 * kC] = v;
          sh.gate[2 * kC + 1] = u;
        }
      }
    }
    cp_wait<0>();
    tc::mbar_wait(&sh.full[0], t & 1, a.err, PL_ERR_MBAR_TIMEOUT);
    {
      F32Tile<DK / 8> ts;
      F32Tile<8> tr;
      ts.take(sh.s[0], tid);
      tr.take(sh.r[t & 1][0], tid);
      __syncthreads();
      ts.template give<LD>(sh.s[0], tid);
      tr.template give<kLd>(sh.r[t & 1][0], tid);
    }
    __syncthreads();
    float x[NK][4];
    zero(x);
    product<false, kLd, 0, true, LD, kState, 4>(x, o, sh.s[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // scale E dO S^T
      const float f = d.since[i0 + half * 8] * a.scale;
#pragma unroll
      for (int n = 0; n < NK; n++) {
        dq[n][half * 2] += f == 0.f ? 0.f : f * x[n][half * 2];
        dq[n][half * 2 + 1] += f == 0.f ? 0.f : f * x[n][half * 2 + 1];
      }
    }
    zero(x);
    product<true, kLd, kRows, true, LD, kState, 4>(x, r, sh.s[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // -E dR S^T
      const float f = -d.since[i0 + half * 8];
#pragma unroll
      for (int n = 0; n < NK; n++) {
        dk[n][half * 2] += f == 0.f ? 0.f : f * x[n][half * 2];
        dk[n][half * 2 + 1] += f == 0.f ? 0.f : f * x[n][half * 2 + 1];
      }
    }
    tc::mbar_wait(&sh.full[1], t & 1, a.err, PL_ERR_MBAR_TIMEOUT);
    F32Tile<DK / 8> ts;
    F32Tile<8> ty;
    ts.take(sh.ds[0], tid);
    ty.take(sh.y[0], tid);
    tc::fence_proxy_async_smem();  // the places of S, dO and dR get new ones
    __syncthreads();
    ts.template give<LD>(sh.ds[0], tid);
    ty.template give<kLd>(sh.y[0], tid);
    if (t + 1 < steps) load_a(t + 1);
    __syncthreads();
    zero(x);
    product<true, kLd, kRows, true, LD, kState, 4>(x, sh.y[0], sh.ds[0], m0, d0);
#pragma unroll
    for (int half = 0; half < 2; half++) {  // F U dS'^T
      const float f = d.until[i0 + half * 8] * d.beta[i0 + half * 8];
#pragma unroll
      for (int n = 0; n < NK; n++) {
        dk[n][half * 2] += f == 0.f ? 0.f : f * x[n][half * 2];
        dk[n][half * 2 + 1] += f == 0.f ? 0.f : f * x[n][half * 2 + 1];
      }
    }
    product<false, kLd, 0, true, kLd, kRows, 4>(oy, o, sh.y[0], m0, n0);
    product<true, kLd, kRows, true, kLd, kRows, 4>(ry, r, sh.y[0], m0, n0);
    tc::fence_proxy_async_smem();
    __syncthreads();
    if (t + 1 < steps) load_b(t + 1);
    if ((t + 1) % slices) continue;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = i0 + half * 8, j = n0 + n * 8 + (lane & 3) * 2, ei = d.era[i];
        const float2 ci = d.cum[i];
        float po[2], mm[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int e = half * 2 + c;
          const float f = j + c <= i ? d.beta[j + c] * decay(ci, ei, d, j + c) : 0.f;
          po[c] = j + c <= i ? a.scale * f * oy[n][e] : 0.f;
          mm[c] = j + c < i ? -f * ry[n][e] : 0.f;
        }
        put2<kLd>(sh.p[0], sh.p[1], i, j, po[0], po[1]);
        put2<kLd>(sh.m[0], sh.m[1], i, j, mm[0], mm[1]);
      }
    __syncthreads();
    product_part<false, kLd, kRows, true, LD, 0>(dq, sh.p[0], sh.k, m0, d0, 0, wr + 1);
    product_part<true, kLd, kRows, true, LD, 0>(dk, sh.p[0], sh.q, m0, d0, wr, 4);
    product_part<false, kLd, kRows, true, LD, 0>(dk, sh.m[0], sh.k, m0, d0, 0, wr + 1);
    product_part<true, kLd, kRows, true, LD, 0>(dk, sh.m[0], sh.k, m0, d0, wr, 4);
    // dbeta, and dg by sums from the chunk's end, cut at resets: by the first warp, for the last head while the others write dq
    // and dk
    auto gates = [&] {
      float sum[2];
      int era[2];
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int i = half * 32 + lane;
        if (i < len) p.dbeta[(start + i) * a.hv + h] = sh.gate[i] / beta_of(d.beta[i]);
        sum[half] = sh.gate[kC + i];
        era[half] = d.era[i];
      }
      const int last = __shfl_sync(0xffffffffu, era[1], 31);
      float behind = sh.gate[2 * kC];  // of the tokens behind this half, as far as they are of era `last`; behind the chunk, <S', dS'>
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
        const int before = __shfl_up_sync(0xffffffffu, era[half], 1), across = __shfl_sync(0xffffffffu, era[0], 31);
        const bool reset = era[half] != (lane ? before : half ? across : 0);
        if (i < len) p.dg[(start + i) * a.hv + h] = reset ? 0.f : i == 0 ? sh.gate[2 * kC + 1] : v;
        behind = __shfl_sync(0xffffffffu, v, 0);
        behind_era = __shfl_sync(0xffffffffu, era[half], 0);
      }
    };
    if (t + 1 < steps) {
      if (warp == 0) gates();
      __syncthreads();
      continue;
    }
    __syncthreads();  // dq and dk leave by way of the places of K and Q, so that rows go out whole
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const int at = (i0 + half * 8) * LD + d0 + n * 8 + (lane & 3) * 2;
        *reinterpret_cast<__nv_bfloat162*>(sh.q + at) = __floats2bfloat162_rn(dq[n][half * 2], dq[n][half * 2 + 1]);
        *reinterpret_cast<__nv_bfloat162*>(sh.k + at) = __floats2bfloat162_rn(dk[n][half * 2], dk[n][half * 2 + 1]);
      }
    __syncthreads();
    if (warp == 0) {
      gates();
      return;
    }
    const long row = (long)a.hk * a.dk, to = start * row + (long)kh * a.dk;
    if (a.dk % 8 == 0 && (((uintptr_t)p.dq | (uintptr_t)p.dk) & 15) == 0) {
      const int pieces = a.dk / 8;
      for (int i = tid - 32; i < len * pieces; i += kGradThreads - 32) {
        const int r = i / pieces, c = i % pieces * 8;
        *reinterpret_cast<uint4*>(p.dq + to + r * row + c) = *reinterpret_cast<const uint4*>(sh.q + r * LD + c);
        *reinterpret_cast<uint4*>(p.dk + to + r * row + c) = *reinterpret_cast<const uint4*>(sh.k + r * LD + c);
      }
    } else {
      for (int i = tid - 32; i < len * a.dk; i += kGradThreads - 32) {
        const int r = i / a.dk, c = i % a.dk;
        p.dq[to + r * row + c] = sh.q[r * LD + c];
        p.dk[to + r * row + c] = sh.k[r * LD + c];
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
static int row_align(const void* p, size_t ld, size_t hs) {
  const uintptr_t all = (uintptr_t)p | ld * 2 | hs * 2;
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
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
  a.dkp = s->dk > 64 ? 128 : 64;
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
  a.err = device_error_word();
  a.vq = row_align(q, s->q_token, s->q_head);
  a.vk = row_align(k, s->k_token, s->k_head);
  a.vv = row_align(v, s->v_token, s->v_head);
  return a;
}
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static size_t heads_slots(const pl_delta_shape* s) {
  return (size_t)slot_count((long)s->tokens, (long)s->sequences) * s->heads_v;
}
static size_t slots_of(const pl_delta_shape* s) { return (size_t)slot_count((long)s->tokens, (long)s->sequences); }
static size_t tiles_bytes(const pl_delta_shape* s) {
  return up256(slots_of(s) * s->heads_k * (s->dk > 64 ? kTileBytes<128> : kTileBytes<64>));
}
// Mats, one behind the other; behind them the tiles of K and Q, and the table of chunks.
static size_t mats_bytes(const pl_delta_shape* s) {
  return up256(heads_slots(s) * sizeof(Mats)) + tiles_bytes(s) + up256(slots_of(s) * sizeof(int2));
}
static __nv_bfloat16* tiles_of(const pl_delta_shape* s, Mats* mats) {
  return (__nv_bfloat16*)((char*)mats + up256(heads_slots(s) * sizeof(Mats)));
}
static int2* table_of(const pl_delta_shape* s, Mats* mats) { return (int2*)((char*)tiles_of(s, mats) + tiles_bytes(s)); }
static size_t states_bytes(const pl_delta_shape* s) {
  return up256(heads_slots(s) * (s->dk > 64 ? 128 : 64) * round_up((long)s->dv, 64) * 4);
}
static size_t lanes_bytes(const pl_delta_shape* s) { return up256(heads_slots(s) * kC * round_up((long)s->dv, 64) * 4); }
static size_t sums_bytes(const pl_delta_shape* s) { return up256(heads_slots(s) * round_up((long)s->dv, 64) / 16 * kSums * 4); }

template <typename A>
static int launch_wide(void (*kernel)(A), dim3 grid, int threads, size_t smem, cudaStream_t st, const A& args) {
  int rc = raise_smem((const void*)kernel, smem);
  if (rc) return rc;
  PL_CUDA(launch_early(kernel, grid, dim3(threads), smem, st, args));
  count_launch();
  return PL_OK;
}
static_assert(sizeof(ScanShared<128>) <= 232448 && sizeof(BackShared<128>) <= 232448 && sizeof(GradShared<128>) <= 232448,
              "shared memory of a block");
static int prep(const DeltaArgs& a, Mats* mats, __nv_bfloat16* tiles, int2* table, cudaStream_t st) {
  const dim3 grid((unsigned)slot_count(a.n, a.seqs), (unsigned)a.hk);
  const bool wide = a.dk > 64;
  const size_t smem = wide ? sizeof(PrepShared<128>) : sizeof(PrepShared<64>);
  auto kernel = wide ? delta_prep_kernel<128> : delta_prep_kernel<64>;
  int rc = raise_smem((const void*)kernel, smem);
  if (rc) return rc;
  PL_CUDA(launch_early(kernel, grid, dim3(kPrepThreads), smem, st, a, mats, tiles, table));
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
  return pl::states_bytes(s) + 2 * pl::lanes_bytes(s) + pl::mats_bytes(s);
}
size_t pl_delta_ws(const pl_delta_shape* s, uint8_t grad) {
  if (!s || s->sequences == 0) return 0;
  const size_t forward = pl::mats_bytes(s), back = pl::states_bytes(s) + pl::lanes_bytes(s) + pl::sums_bytes(s);
  return !grad ? forward : (back > forward ? back : forward) + 256;  // the gradient's serves the forward call, too
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
  PL_REQUIRE(saved || (ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= pl_delta_ws(s, 0)), PL_ERR_INVALID,
             "%s: %zu bytes of workspace at 256 bytes needed", me, pl_delta_ws(s, 0));
  PL_REQUIRE(!saved || ((uintptr_t)saved % 256 == 0 && saved_bytes >= pl_delta_saved(s)), PL_ERR_INVALID,
             "%s: %zu bytes at 256 bytes needed for the gradient's states", me, pl_delta_saved(s));
  rc = require_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const DeltaArgs a = delta_args(s, q, k, v, g, beta, offsets);
  Mats* mats = (Mats*)(saved ? (char*)saved + states_bytes(s) + 2 * lanes_bytes(s) : ws);
  if (s->tokens) {
    rc = prep(a, mats, tiles_of(s, mats), table_of(s, mats), st);
    if (rc) return rc;
  }
  ScanArgs p = {a, mats, tiles_of(s, mats), state, (__nv_bfloat16*)o, final_state, nullptr, nullptr, nullptr};
  if (saved) {
    p.kept = (float*)saved;
    p.y = (float*)((char*)saved + states_bytes(s));
    p.out = (float*)((char*)saved + states_bytes(s) + lanes_bytes(s));
  }
  const dim3 grid((unsigned)(a.dvp / 64), (unsigned)a.hv, (unsigned)a.seqs);
  auto kernel = saved ? (a.dk > 64 ? delta_scan_kernel<128, true> : delta_scan_kernel<64, true>)
                      : (a.dk > 64 ? delta_scan_kernel<128, false> : delta_scan_kernel<64, false>);
  return launch_wide(kernel, grid, kChainThreads, a.dk > 64 ? sizeof(ScanShared<128>) : sizeof(ScanShared<64>), st, p);
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
  float *ds = (float*)ws, *dr = (float*)((char*)ws + states_bytes(s)), *sums = (float*)((char*)dr + lanes_bytes(s));
  const float *kept = (const float*)saved, *y = (const float*)((const char*)saved + states_bytes(s));
  const float* out = (const float*)((const char*)y + lanes_bytes(s));
  const int align_o = row_align(dout, do_token, do_head);
  Mats* mats = (Mats*)((char*)out + lanes_bytes(s));
  const BackArgs b = {a, mats, tiles_of(s, mats), (const __nv_bfloat16*)dout, (long)do_token, (long)do_head, align_o, dfinal,
                      kept, y, out, (__nv_bfloat16*)dv, dstate, ds, dr, sums};
  const dim3 grid((unsigned)(a.dvp / 64), (unsigned)a.hv, (unsigned)a.seqs);
  rc = a.dk > 64 ? launch_wide(delta_back_kernel<128>, grid, kChainThreads, sizeof(BackShared<128>), st, b)
                 : launch_wide(delta_back_kernel<64>, grid, kChainThreads, sizeof(BackShared<64>), st, b);
  if (rc || s->tokens == 0) return rc;
  const GradArgs p = {a, (const __nv_bfloat16*)dout, (long)do_token, (long)do_head, align_o, kept, y, ds, dr, sums, mats,
                      tiles_of(s, mats), table_of(s, mats), (__nv_bfloat16*)dq, (__nv_bfloat16*)dk, dg, dbeta};
  const dim3 chunks((unsigned)slot_count(a.n, a.seqs), (unsigned)a.hk);
  rc = a.dk > 64 ? launch_wide(delta_grad_kernel<128>, chunks, kGradThreads, sizeof(GradShared<128>), st, p)
                 : launch_wide(delta_grad_kernel<64>, chunks, kGradThreads, sizeof(GradShared<64>), st, p);
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
