// What the kernels of the gated delta rule share: the cut of packed sequences into chunks of 64 tokens, copies of tiles
// into shared memory, and products of bf16 tiles whose f32 operands are carried as two or three bf16 parts.
#pragma once
#include <type_traits>

#include "pl_common.cuh"
#include "pl_tc.cuh"

namespace pl {

constexpr int kC = 64;    // tokens of a chunk
constexpr int kLd = 72;   // row stride of a 64-column bf16 tile in shared memory: rows 16 bytes apart in the banks

struct DeltaArgs {
  long n;                      // tokens
  int seqs, hk, hv, dk, dv, dkp, dvp;  // dkp: 64 or 128; dvp: dv rounded up to 64
  const int* offsets;          // [seqs + 1], or NULL: sequences of n / seqs tokens
  long ldq, hsq, ldk, hsk, ldv, hsv;  // strides of tokens and heads
  const __nv_bfloat16 *q, *k, *v;
  const float *g, *beta;  // [n][hv]
  float scale;
  unsigned* err;  // where a wait for copies that ran out is recorded
  int vq, vk, vv;  // bytes (16, 8, 4, 2) at whose multiples all rows of q, k, v start
};

// Sequence s's tokens, whatever the offsets hold: inside [0, n].
__device__ __forceinline__ void seq_bounds(const DeltaArgs& a, int s, long& from, long& to) {
  if (a.offsets) {
    from = a.offsets[s];
    to = a.offsets[s + 1];
  } else {
    from = a.n / a.seqs * s;
    to = from + a.n / a.seqs;
  }
  from = from < 0 ? 0 : from > a.n ? a.n : from;
  to = to < from ? from : to > a.n ? a.n : to;
}
// Chunk c of sequence s has slot from / 64 + s + c: no two share one (a sequence of L tokens has at most L / 64 + 1
// chunks, and the next one's first slot is at least that much further), and all are below n / 64 + seqs.
__device__ __forceinline__ long seq_slot(const DeltaArgs& a, int s) {
  long from, to;
  seq_bounds(a, s, from, to);
  return from / kC + s;
}
__host__ __device__ __forceinline__ long slot_count(long n, long seqs) { return n / kC + seqs; }

// The chunk of a slot: its first token and how many it has (0: none). By whole warps, 32 sequences at a time: one after the
// other, the reads of a binary search took longer than what the kernels do with the answer.
__device__ __forceinline__ int slot_chunk(const DeltaArgs& a, long slot, long& start) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.seqs;  // the last sequence whose first slot is not behind this one: in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32, s = lo + lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, lane * step < n && seq_slot(a, s) <= slot);
    const int last = m ? 31 - __clz(m) : 0;
    lo += last * step;
    n = n - last * step < step ? n - last * step : step;
  }
  long from, to;
  seq_bounds(a, lo, from, to);
  start = from + (slot - from / kC - lo) * kC;
  if (start < from || start >= to) return 0;
  return (int)(to - start < kC ? to - start : kC);
}

using tc::smem_u32;
__device__ __forceinline__ void cp16(void* dst, const void* src, int bytes) {  // the rest of the 16 bytes is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void cp_few(void* dst, const void* src, int bytes) {  // BYTES 4 or 8
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES), "r"(bytes)
               : "memory");
}
// 64 rows x COLS values into a tile of row stride LD, from rows of `stride`; what is outside rows x cols becomes zero. `align`:
// the bytes at whose multiples the rows start; at 2, values are copied one by one, otherwise asynchronously (cp_commit,
// cp_wait).
template <int COLS, int LD, int THREADS>
__device__ __forceinline__ void copy_tile(__nv_bfloat16* dst, const __nv_bfloat16* src, long stride, int rows, int cols,
                                          int align, int tid) {
  auto pieces = [&](auto piece) {
    constexpr int BYTES = decltype(piece)::value, N = BYTES / 2;
#pragma unroll 4
    for (int i = tid; i < kC * (COLS / N); i += THREADS) {
      const int r = i / (COLS / N), c = i % (COLS / N) * N;
      int bytes = r < rows ? (cols - c) * 2 : 0;
      bytes = bytes < 0 ? 0 : bytes > BYTES ? BYTES : bytes;
      const __nv_bfloat16* from = bytes ? src + (long)r * stride + c : src;
      if constexpr (BYTES == 16) cp16(dst + r * LD + c, from, bytes);
      else cp_few<BYTES>(dst + r * LD + c, from, bytes);
    }
  };
  if (align >= 16) {
    pieces(std::integral_constant<int, 16>());
  } else if (align == 8) {
    pieces(std::integral_constant<int, 8>());
  } else if (align == 4) {
    pieces(std::integral_constant<int, 4>());
  } else {
#pragma unroll 8
    for (int i = tid; i < kC * COLS; i += THREADS) {
      const int r = i / COLS, c = i % COLS;
      dst[r * LD + c] = r < rows && c < cols ? src[(long)r * stride + c] : __float2bfloat16_rn(0.f);
    }
  }
}
// Bulk copies: 16-byte aligned addresses, a multiple of 16 bytes; into shared memory `bar` counts the bytes that are there, out
// of it the thread waits by bulk_read. One instruction of one thread, and no traffic through the load and store units,
// which asynchronous copies of 16 bytes kept busy for a third of a chunk's time. (Row by row, 192 of them per chunk, they
// were slower than those.)
__device__ __forceinline__ void bulk_in(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

// ---------------------------------------------------------------------------------------------- products
// m16n8k16 products of one warp on bf16 tiles in shared memory. An operand lies either along k (rows of m or n) or
// across it (rows of k); ldmatrix transposes the latter.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where this lane's rows of the 16 x 16 fragment at (0, 0) of an operand start, in elements: of A, along k or across, and of two
// n-tiles of B (registers 0, 1 for the columns from n on, 2, 3 for n + 8).
template <bool ACROSS, int LD>
__device__ __forceinline__ int lane_a() {
  const int lane = threadIdx.x & 31;
  if constexpr (!ACROSS) return (lane & 15) * LD + (lane >> 4) * 8;
  else return ((lane & 7) + ((lane >> 4) & 1) * 8) * LD + ((lane >> 3) & 1) * 8;
}
template <bool ACROSS, int LD>
__device__ __forceinline__ int lane_b() {
  const int lane = threadIdx.x & 31;
  if constexpr (!ACROSS) return ((lane & 7) + ((lane >> 4) & 1) * 8) * LD + ((lane >> 3) & 1) * 8;
  else return ((lane & 7) + ((lane >> 3) & 1) * 8) * LD + ((lane >> 4) & 1) * 8;
}
template <bool ACROSS>
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
  if constexpr (ACROSS) ldsm4t(r, at);
  else ldsm4(r, at);
}

// acc (16 x 8 NT at (m, n)) += A B over KS steps of 16 along k, from tile rows and columns (m, k = 0), (k = 0, n) on. A f32
// operand is two bf16 parts, the second one the rounding of what the first leaves, ALO or BLO elements behind it (2^-17 of the
// value is lost, the product of the two second parts with it); 0: bf16 as it is. Addresses are one register and constants.
template <bool A_ACROSS, int LDA, int ALO, bool B_ACROSS, int LDB, int BLO, int KS, int NT>
__device__ __forceinline__ void product(float (&acc)[NT][4], const __nv_bfloat16* a, const __nv_bfloat16* b, int m, int n) {
  const uint32_t pa = smem_u32(a + (A_ACROSS ? m : m * LDA) + lane_a<A_ACROSS, LDA>());
  const uint32_t pb = smem_u32(b + (B_ACROSS ? n : n * LDB) + lane_b<B_ACROSS, LDB>());
#pragma unroll
  for (int k = 0; k < KS; k++) {
    uint32_t x[4], xl[4];
    ldsm<A_ACROSS>(x, pa + k * 32 * (A_ACROSS ? LDA : 1));
    if constexpr (ALO != 0) ldsm<A_ACROSS>(xl, pa + ALO * 2 + k * 32 * (A_ACROSS ? LDA : 1));
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      uint32_t y[4];
      const uint32_t at = pb + k * 32 * (B_ACROSS ? LDB : 1) + t * 16 * (B_ACROSS ? 1 : LDB);
      ldsm<B_ACROSS>(y, at);
      mma(acc[t], x, y[0], y[1]);
      mma(acc[t + 1], x, y[2], y[3]);
      if constexpr (ALO != 0) {
        mma(acc[t], xl, y[0], y[1]);
        mma(acc[t + 1], xl, y[2], y[3]);
      }
      if constexpr (BLO != 0) {
        ldsm<B_ACROSS>(y, at + BLO * 2);
        mma(acc[t], x, y[0], y[1]);
        mma(acc[t + 1], x, y[2], y[3]);
      }
    }
  }
}
// The same over the row blocks [k0, k1) of k.
template <bool A_ACROSS, int LDA, int ALO, bool B_ACROSS, int LDB, int BLO, int NT>
__device__ __forceinline__ void product_part(float (&acc)[NT][4], const __nv_bfloat16* a, const __nv_bfloat16* b, int m,
                                             int n, int k0, int k1) {
  for (int k = k0; k < k1; k++)
    product<A_ACROSS, LDA, ALO, B_ACROSS, LDB, BLO, 1>(acc, a + k * 16 * (A_ACROSS ? LDA : 1),
                                                       b + k * 16 * (B_ACROSS ? LDB : 1), m, n);
}

// A lower triangular 64 x 64 matrix as the ten 16 x 16 blocks on and below its diagonal, block (r, c) the r (r + 1) / 2 + c-th;
// in a block, row i's two 16-byte pieces change places where i & 4, so that ldmatrix's eight rows are in eight places.
constexpr int kTri = 10 * 256;
__host__ __device__ __forceinline__ int tri_at(int i, int j) {
  const int r = i >> 4, c = j >> 4, y = i & 15, x = j & 15;
  return (r * (r + 1) / 2 + c) * 256 + y * 16 + (((x >> 3) ^ ((y >> 2) & 1)) << 3) + (x & 7);
}
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// A fragment's pair of values at (row, col) of a tile, as two parts.
template <int LD>
__device__ __forceinline__ void put2(__nv_bfloat16* hi, __nv_bfloat16* lo, int row, int col, float x, float y) {
  uint32_t h, l;
  split2(x, y, h, l);
  *reinterpret_cast<uint32_t*>(hi + row * LD + col) = h;
  *reinterpret_cast<uint32_t*>(lo + row * LD + col) = l;
}

// ---- products whose first operand is in registers: an accumulator's two neighbouring n-tiles, 16 rows x 16 columns, are
// the fragment of A for 16 steps of k, as N bf16 parts: three hold all 24 bits of an f32.
template <int N>
struct Parts {
  uint32_t p[N][4];
};
template <int N>
__device__ __forceinline__ void split(float x, float y, Parts<N>& to, int at) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    to.p[i][at] = *reinterpret_cast<const uint32_t*>(&h);
    x -= __low2float(h);
    y -= __high2float(h);
  }
}
template <int N>
__device__ __forceinline__ Parts<N> parts_of(const float (&x)[4], const float (&y)[4]) {
  Parts<N> r;
  split<N>(x[0], x[1], r, 0);
  split<N>(x[2], x[3], r, 1);
  split<N>(y[0], y[1], r, 2);
  split<N>(y[2], y[3], r, 3);
  return r;
}
// acc [16][16 N] += A B for one 16 of k: B bf16, at `at` and every `step` bytes. The first parts add to `acc` and the others to `low`,
// which joins it by `join`: the tensor cores cut a sum off behind its 24th bit, towards zero, and a small product added to a large
// sum costs it as much as a large one. All first parts go before the second ones: a product waits 25 cycles for the one before
// it on the same accumulator, and N of them take 8 N.
template <bool ACROSS, int N, int PARTS>
__device__ __forceinline__ void step(float (&acc)[2 * N][4], float (&low)[2 * N][4], const Parts<PARTS>& a, uint32_t at,
                                     int step) {
  uint32_t y[N][4];
#pragma unroll
  for (int n = 0; n < N; n++) ldsm<ACROSS>(y[n], at + n * step);
#pragma unroll
  for (int i = 0; i < PARTS; i++)
#pragma unroll
    for (int n = 0; n < N; n++) {
      mma(i ? low[2 * n] : acc[2 * n], a.p[i], y[n][0], y[n][1]);
      mma(i ? low[2 * n + 1] : acc[2 * n + 1], a.p[i], y[n][2], y[n][3]);
    }
}
template <int NT>
__device__ __forceinline__ void join(float (&acc)[NT][4], const float (&low)[NT][4]) {
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[t][e] += low[t][e];
}
// to(t, sum) for the n-tiles t of A B over the four 16 of a chunk's tokens, [16][8 NT], B across; half of them at a time, so that
// the sums of parts have registers.
template <int LD, int NT, int PARTS, typename F>
__device__ __forceinline__ void token_steps(const Parts<PARTS> (&a)[4], uint32_t at, F to) {
#pragma unroll
  for (int q = 0; q < 2; q++) {
    float acc[NT / 2][4], low[NT / 2][4];
#pragma unroll
    for (int t = 0; t < NT / 2; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[t][e] = low[t][e] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) step<true, NT / 4>(acc, low, a[k], at + k * 32 * LD + q * NT * 8, 32);
    join(acc, low);
#pragma unroll
    for (int t = 0; t < NT / 2; t++) to(q * (NT / 2) + t, acc[t]);
  }
}
// acc [dv][64 tokens] += A T^T (ACROSS = false: column block n over blocks k <= n) or A T (ACROSS: over k >= n) for A's four 16
// columns; T triangular, three parts. Of parts i and j, those with i + j < PAIRS, the smallest products first.
template <bool ACROSS, int PARTS, int PAIRS>
__device__ __forceinline__ void tri_product(float (&acc)[8][4], const Parts<PARTS> (&a)[4], uint32_t tri) {
#pragma unroll
  for (int ij = PAIRS - 1; ij >= 0; ij--)
#pragma unroll
    for (int j = 0; j <= ij; j++) {
      const int i = ij - j;
      if (i >= PARTS) continue;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        uint32_t y[4][4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
          if (ACROSS ? n > k : n < k) continue;
          const int r = ACROSS ? k : n, c = ACROSS ? n : k;
          ldsm<ACROSS>(y[n], tri + (r * (r + 1) / 2 + c) * 512 + j * kTri * 2);
        }
#pragma unroll
        for (int n = 0; n < 4; n++) {
          if (ACROSS ? n > k : n < k) continue;
          mma(acc[2 * n], a[k].p[i], y[n][0], y[n][1]);
          mma(acc[2 * n + 1], a[k].p[i], y[n][2], y[n][3]);
        }
      }
    }
}
// Registers of one warp for another one's same lanes: pieces of 16 bytes per lane at `at`.
__device__ __forceinline__ void give(uint4* at, int piece, const uint32_t (&r)[4]) {
  at[piece * 32 + (threadIdx.x & 31)] = make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ void give(uint4* at, int piece, const float (&r)[4]) {
  at[piece * 32 + (threadIdx.x & 31)] =
      make_uint4(__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3]));
}
__device__ __forceinline__ void take(const uint4* at, int piece, uint32_t (&r)[4]) {
  const uint4 v = at[piece * 32 + (threadIdx.x & 31)];
  r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
}
__device__ __forceinline__ void take(const uint4* at, int piece, float (&r)[4]) {
  const uint4 v = at[piece * 32 + (threadIdx.x & 31)];
  r[0] = __uint_as_float(v.x), r[1] = __uint_as_float(v.y), r[2] = __uint_as_float(v.z), r[3] = __uint_as_float(v.w);
}
// Barrier `id` of THREADS threads: what those that arrive wrote before, those that wait see behind it. Each of them comes once
// before any comes again, by one or the other.
template <int THREADS>
__device__ __forceinline__ void meet_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void meet(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}

// This lane's place in a triangular matrix's first block as B: [n][k] as it lies, or (ACROSS) [k][n].
template <bool ACROSS>
__device__ __forceinline__ uint32_t tri_lane(const __nv_bfloat16* t) {
  const int lane = threadIdx.x & 31;
  const int y = (lane & 7) + ((ACROSS ? lane >> 3 : lane >> 4) & 1) * 8, p = (ACROSS ? lane >> 4 : lane >> 3) & 1;
  return smem_u32(t + y * 16 + ((p ^ ((y >> 2) & 1)) << 3));
}
// Four 8 x 8 blocks of an accumulator [dv][token] into rows of tokens: n-tiles t and t + 1, 16 values of every token.
__device__ __forceinline__ void store_across(uint32_t at, const float (&x)[4], const float (&y)[4]) {
  const __nv_bfloat162 v[4] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3]),
                               __floats2bfloat162_rn(y[0], y[1]), __floats2bfloat162_rn(y[2], y[3])};
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}

template <int NT>
__device__ __forceinline__ void zero(float (&acc)[NT][4]) {
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[t][e] = 0.f;
}

// The decays of a chunk's tokens, by the block's first warp: cum (sum of g / ln 2 since the last reset or the chunk's start, in
// f64 and kept as two f32, so that differences of large sums are right), era (resets so far), since = the factor on
// the state before the chunk (zero behind a reset), until = the factor from a token to the chunk's end (zero in front of a
// reset). A g of -inf resets, and so does one below -104, whose factor f32 cannot hold.
struct __align__(16) Decay {
  float2 cum[kC];
  int era[kC];
  float since[kC], until[kC], beta[kC];
};
__device__ __forceinline__ float exp2_of(float x) {  // 2^-22 off; zero below 2^-126
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
// The same of an f64 exponent: what its f32 leaves, up to 4e-6 of the result far below zero, is multiplied in.
__device__ __forceinline__ float exp2_of(double x) {
  const float hi = (float)x;
  return exp2_of(hi) * __fmaf_rn((float)(x - (double)hi), 0.69314718f, 1.f);
}
struct Gates {
  float g[2], beta[2];  // of tokens lane and lane + 32, in the block's first warp
};
__device__ __forceinline__ Gates load_gates(const DeltaArgs& a, long start, int len, int h) {
  Gates r;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int t = half * 32 + threadIdx.x;
    const bool in = threadIdx.x < 32 && t < len;
    r.g[half] = in ? a.g[(start + t) * a.hv + h] : 0.f;
    r.beta[half] = in ? a.beta[(start + t) * a.hv + h] : 0.f;
  }
  return r;
}
__device__ __forceinline__ void chunk_decay(Decay& d, const Gates& r) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    double cum[2];
    int era[2];
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int t = half * 32 + lane;
      const float g = r.g[half];
      d.beta[t] = r.beta[half];
      const bool reset = g < -104.f;
      cum[half] = reset ? 0.0 : (double)g * 1.4426950408889634074;
      era[half] = reset;
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2)  // (sum, resets) of the tokens up to this one; a reset forgets the sum before it
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const double up = __shfl_up_sync(0xffffffffu, cum[half], o);
        const int ue = __shfl_up_sync(0xffffffffu, era[half], o);
        if (lane >= o) {
          if (era[half] == 0) cum[half] += up;
          era[half] += ue;
        }
      }
    const double first = __shfl_sync(0xffffffffu, cum[0], 31);
    if (era[1] == 0) cum[1] += first;
    era[1] += __shfl_sync(0xffffffffu, era[0], 31);
    const double end = __shfl_sync(0xffffffffu, cum[1], 31);
    const int last = __shfl_sync(0xffffffffu, era[1], 31);
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int t = half * 32 + lane;
      const float hi = (float)cum[half];
      d.cum[t] = make_float2(hi, (float)(cum[half] - (double)hi));
      d.era[t] = era[half];
      d.since[t] = era[half] == 0 ? exp2_of(cum[half]) : 0.f;
      d.until[t] = era[half] == last ? exp2_of(end - cum[half]) : 0.f;
    }
  }
}
// The factor from token j to token i >= j.
__device__ __forceinline__ float decay(float2 ci, int ei, const Decay& d, int j) {
  const float2 cj = d.cum[j];
  return ei == d.era[j] ? exp2_of((ci.x - cj.x) + (ci.y - cj.y)) : 0.f;
}

}  // namespace pl
