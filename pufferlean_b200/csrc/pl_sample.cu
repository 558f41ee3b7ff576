// Drawing tokens from logits with temperature, top-k, top-p and min-p, one given uniform number per row.
//
//   e_i = exp((z_i - max z) / T);  order: larger z first, among equals the lower index first
//   kept = the first k in order; of these those before which less than p of their mass comes; of these those with
//          e_i >= min_p. The first in order always stays.
//   token = the first kept i, by index, with sum_{kept j <= i} e_j > u sum_kept e;  logp = log(e_token / sum_kept e)
//
// Every sum is f64, and so is every exponential behind one: a row of V near-equal tokens has V borders, and f32 sums
// (1e-7 off) would move one of them across u in 2 rows of 100 at V = 131,072.
//
// Many rows, and short ones: a CTA per row, which walks it from L2 for each step below (the rows in flight fit there). Few long
// rows: a cluster of CTAs per row, each with a contiguous slice in shared memory.
//
// Without filters that is one walk with f64 sums by warp, segment and lane; the segment of u's place is walked once more.
// The border of top-k or top-p is found in three steps. (1) A sample of the row and a walk with f32 weights put counts or
// masses into 64 bins of d = ref - z, each thread's its own (no atomics): this proposes an interval [zb, za] of logits
// around the border. (2) A walk in f64 takes the masses above, in and below the interval and lists what lies in it. (3) If
// these say that the border is inside, which they do but for a few rows in a million, the list is sorted and the border
// is exact. If the proposal fails, more walks propose; if the list overflows (more equal logits than it holds), the
// border's key is searched bit by bit. So sample and f32 sums cost time where they are off, never a token. top_k up to 1,024
// takes one walk: the sample gives a bound that surely more than k pass, and what passes it is listed and sorted.
//
// Exponents refer to the sample's largest logit instead of the row's: f64 has the room (2^900), and the walk that needs it
// finds the largest on its way.
//
// Bound by instructions: the f64 walk is 45 per 32 logits (12 of them f64, 6 clocks of an SM's f64 pipe), the f32 walk 20, at
// half an instruction per clock and scheduler. 1,024 x 131,072 bf16: 249 us without filters, 630 to 670 with top_p 0.9,
// 174 with top_k 50 (HBM: 41); 2,047 x 50,021 f32 249 (63).
#include <cooperative_groups.h>

#include <type_traits>

#include "pl_common.cuh"
#include "pl_runtime.h"

namespace cg = cooperative_groups;

namespace pl {

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 64, kList = 2048, kSegs = 16;
constexpr int kMostVocab = 1 << 18;
constexpr double kLeastTemp = 1e-38, kMostTemp = 1e30;  // a temperature beyond counts as these

struct SampleArgs {
  const void* logits;
  long ld;
  int V, slice;  // slice: values of a row per CTA, a multiple of 8
  const float *u, *temp, *p, *min_p;  // temp, p, min_p, k: one per row, or NULL: the number below
  const int* k;
  double temp0, p0, min_p0;
  int k0;
  int* token;
  float* logp;
};

// An unsigned key that orders like the value; both zeros have one key.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float exp2_fast(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return e;
}

__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}

// An f32 times 2^-896 as a double, by moving its bits (a conversion has a quarter of the rate): with the exponent's field as it
// is, zeros and numbers below the smallest normal one are exact as well. -inf is -2^128.
__device__ __forceinline__ double moved(float z) {
  const uint32_t b = __float_as_uint(z);
  return __hiloint2double((int)((b & 0x80000000u) | ((b & 0x7fffffffu) >> 3)), (int)(b << 29));
}

// exp((z - ref) / T) in f64: 2^y, y = n / 16 + r with 2^(n / 16) from a table and 2^r, |r| <= 1/32, from five terms of its series
// (the sixth is 1.4e-13 of the value at most). Both are moved alike, so that y is exactly zero for equal logits, whatever T.
struct Exp {
  double ref, c;  // ref 2^-896, log2(e) / T 2^896 (T >= kLeastTemp: below 2^1023)
  const double* tab;
  // N values step by step side by side: one after the other, each waits out the latency of a dozen f64 operations.
  template <int N>
  __device__ __forceinline__ void many(const float* z, double* e) const {
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
    const double l = 0.6931471805599453094;
    double y[N], s[N], q[N];
    int n[N];
    bool in[N];
#pragma unroll
    for (int j = 0; j < N; j++) y[j] = moved(z[j]) - ref;
#pragma unroll
    for (int j = 0; j < N; j++) y[j] *= c;
#pragma unroll
    for (int j = 0; j < N; j++) {
      in[j] = (uint32_t)__double2hiint(y[j]) < 0xc08f4000u;  // y > -1000: by the order of negative doubles' bits
      s[j] = fma(y[j], 16.0, magic);
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      n[j] = __double2loint(s[j]);
      s[j] -= magic;
    }
#pragma unroll
    for (int j = 0; j < N; j++) y[j] = fma(s[j], -0.0625, y[j]);
    const double k5 = l * l * l * l * l / 120.0, k4 = l * l * l * l / 24.0, k3 = l * l * l / 6.0, k2 = l * l / 2.0;
#pragma unroll
    for (int j = 0; j < N; j++) q[j] = fma(k5, y[j], k4);
#pragma unroll
    for (int j = 0; j < N; j++) q[j] = fma(q[j], y[j], k3);
#pragma unroll
    for (int j = 0; j < N; j++) q[j] = fma(q[j], y[j], k2);
#pragma unroll
    for (int j = 0; j < N; j++) q[j] = fma(q[j], y[j], l);
#pragma unroll
    for (int j = 0; j < N; j++) q[j] = fma(q[j], y[j], 1.0);
#pragma unroll
    for (int j = 0; j < N; j++) q[j] *= tab[n[j] & 15];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const double x = __hiloint2double(__double2hiint(q[j]) + (n[j] >> 4) * (1 << 20), __double2loint(q[j]));
      e[j] = in[j] ? x : 0.0;
    }
  }
  __device__ __forceinline__ double operator()(float z) const {
    double e;
    many<1>(&z, &e);
    return e;
  }
};

struct Shared {
  double x[2][kBins];  // what the cluster's CTAs read of one another, by turns
  double warp[kWarps][4];
  double seg[kWarps * kSegs];
  double tab[16];
  float fwarp[kWarps][4];
  int iwarp[kWarps];
  int count, found;
  float tz;
  uint32_t tidx;
  unsigned char part[kList];
};

// SOLO: the block has the whole row and reads it from memory; otherwise a cluster, each block with a slice in shared
// memory.
template <typename T, bool SOLO>
__global__ void __launch_bounds__(kThreads, SOLO ? 3 : 2) sample_kernel(const SampleArgs a) {
  grid_wait();
  grid_next();
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char mem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = SOLO ? 1 : (int)cluster.num_blocks(), rank = SOLO ? 0 : (int)cluster.block_rank();
  auto sync = [&] {
    if constexpr (SOLO) __syncthreads();
    else cluster.sync();
  };
  auto of_rank = [&](auto* p, int q) {
    if constexpr (SOLO) return p;
    else return cluster.map_shared_rank(p, q);
  };
  const long row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // 64 KB by turns: bins [kBins][kThreads] f32; or rank 0's list, sums by warp, segment and lane, and the list's masses
  float* hist = reinterpret_cast<float*>(mem);
  unsigned long long* list = reinterpret_cast<unsigned long long*>(mem);
  double* sub = reinterpret_cast<double*>(mem + 8 * kList);
  double* list_e = reinterpret_cast<double*>(mem + 8 * kList + 8 * kThreads * kSegs);
  static_assert(8 * kList * 2 + 8 * kThreads * kSegs <= 4 * kBins * kThreads, "parts of the work area");
  T* cache = reinterpret_cast<T*>(mem + sizeof(float) * kBins * kThreads);

  // ---- the row's options
  const double t_given = a.temp ? (double)a.temp[row] : a.temp0, p_given = a.p ? (double)a.p[row] : a.p0;
  const double mp_given = a.min_p ? (double)a.min_p[row] : a.min_p0;
  const double u_given = (double)a.u[row];
  int k = a.k ? a.k[row] : a.k0;
  double temp = fmin(t_given, kMostTemp), top_p = p_given, min_p = fmin(mp_given, 1.0);
  const double u = fmin(fmax(u_given, 0.0), 1.0);
  const bool fine = t_given >= 0.0 && t_given < INFINITY && p_given == p_given && mp_given == mp_given && u_given == u_given;
  if (temp == 0.0 || top_p <= 0.0) k = 1;  // the first in order alone
  if (k == 1) {
    temp = 1.0;
    top_p = 1.0;
    min_p = 0.0;
  }
  temp = fmax(temp, kLeastTemp);
  if (k <= 0 || k >= a.V) k = 0;

  // ---- the slice: vectors of 16 bytes at 16-byte boundaries, a warp's together; around it -inf
  const long first = (long)rank * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  const int len = last > first ? (int)(last - first) : 0;
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + first;
  const int shift = len ? (int)(((uintptr_t)src & 15) / sizeof(T)) : 0;
  const int vecs = (shift + len + VEC - 1) / VEC;
  const int its = (vecs + kThreads - 1) / kThreads, per_warp = its * 32;  // iterations, vectors of a warp
  auto fetch = [&](int v) {
    uint4 w;
    const int at = v * VEC - shift;
    if (at >= 0 && at + VEC <= len) return __ldg(reinterpret_cast<const uint4*>(src + at));
    T x[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) x[j] = at + j >= 0 && at + j < len ? src[at + j] : (T)(-INFINITY);
    memcpy(&w, x, 16);
    return w;
  };
  auto value = [&](const uint4& w, int j) {
    const uint32_t u4[4] = {w.x, w.y, w.z, w.w};
    if constexpr (VEC == 4) return __uint_as_float(u4[j]);
    else return __uint_as_float(j & 1 ? u4[j / 2] & 0xffff0000u : u4[j / 2] << 16);
  };
  // f(VEC values, the first one's index in the row) for the vectors of warp w's iterations [i0, i1), and done(iteration)
  // behind each; U vectors are loaded at a time. What f computes of all values before it branches on one of them overlaps.
  auto walk_part = [&](auto unroll, int w, int i0, int i1, auto f, auto done) {
    constexpr int U = decltype(unroll)::value;
    for (int it = i0; it < i1; it += U) {
      uint4 x[U];
      const int v0 = w * per_warp + it * 32;  // the warp's first vector
      if (SOLO && it + U <= i1 && v0 * VEC >= shift && (v0 + 32 * U) * VEC - shift <= len) {
        const uint4* at = reinterpret_cast<const uint4*>(src - shift) + v0 + lane;
#pragma unroll
        for (int q = 0; q < U; q++) x[q] = __ldg(at + 32 * q);
      } else {
#pragma unroll
        for (int q = 0; q < U; q++) {
          const int v = v0 + q * 32 + lane;
          if (it + q < i1 && v < vecs) {
            if constexpr (SOLO) x[q] = fetch(v);
            else x[q] = *reinterpret_cast<const uint4*>(cache + v * VEC);
          } else {
            const uint32_t none = VEC == 4 ? 0xff800000u : 0xff80ff80u;
            x[q] = make_uint4(none, none, none, none);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < U; q++) {
        const uint32_t i = (uint32_t)(first + (v0 + q * 32 + lane) * VEC - shift);
        float z[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) z[j] = value(x[q], j);
        f(z, i);
        if (it + q < i1) done(it + q);
      }
    }
  };
  auto nothing = [](int) {};
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  using ByCount = std::false_type;
  using ByMass = std::true_type;

  // ---- a sample of the slice (all of it, if it is short), and its largest logit as what exponents refer to: any logit
  // not far below the largest will do, and the walks below find the largest on their way
  if constexpr (!SOLO) {
    for (int it = 0; it < its; it++) {
      const int v = warp * per_warp + it * 32 + lane;
      if (v < vecs) *reinterpret_cast<uint4*>(cache + v * VEC) = fetch(v);
    }
    __syncthreads();
  }
  constexpr int kSample = 4;  // vectors per thread
  const int sampled = vecs < kSample * kThreads ? vecs : kSample * kThreads;
  auto walk_sample = [&](auto f) {
    uint4 x[kSample];
#pragma unroll
    for (int q = 0; q < kSample; q++) {
      const int n = q * kThreads + tid;
      const uint32_t none = VEC == 4 ? 0xff800000u : 0xff80ff80u;
      x[q] = make_uint4(none, none, none, none);
      if (n < sampled) {
        const int v = vecs <= kSample * kThreads ? n : (int)((long)n * vecs / (kSample * kThreads));
        if constexpr (SOLO) x[q] = fetch(v);
        else x[q] = *reinterpret_cast<const uint4*>(cache + v * VEC);
      }
    }
#pragma unroll
    for (int q = 0; q < kSample; q++) {
      float z[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) z[j] = value(x[q], j);
      f(z, 0u);
    }
  };
  auto largest = [&](const float (&z)[VEC], float m) {
#pragma unroll
    for (int j = 0; j < VEC; j++) m = max_nan(m, z[j]);
    return m;
  };
  if (tid < 16) sh.tab[tid] = exp2((double)tid / 16.0);
  if (tid == 0) sh.count = 0;
  // The largest of the cluster's numbers, NaN if one of them is.
  auto max_of_all = [&](float m) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh.fwarp[warp][0] = m;
    sync();
    for (int q = 0; q < ranks; q++) {
      const float* other = of_rank(&sh.fwarp[0][0], q);
      for (int w = 0; w < kWarps; w++) m = max_nan(m, other[4 * w]);
    }
    sync();
    return m;
  };
  float ref = -INFINITY;
  walk_sample([&](const float(&z)[VEC], uint32_t) { ref = largest(z, ref); });
  ref = max_of_all(ref);
  float top = ref;  // the largest logit, once a walk over all of them is done
  auto walk_max = [&]() __attribute__((always_inline)) {
    float m = -INFINITY;
    walk_part(Four(), warp, 0, its, [&](const float(&z)[VEC], uint32_t) { m = largest(z, m); }, nothing);
    top = max_of_all(m);
  };
  const bool plain = k == 0 && top_p >= 1.0 && min_p <= 0.0;
  const bool few = k > 0 && k <= kList / 2, nucleus = k == 0 && top_p < 1.0;
  bool known = false;  // whether `top` is of all
  if (ref == -INFINITY || !(plain || few || nucleus)) {
    walk_max();
    ref = top;
    known = true;
  }
  auto bad = [&](float z) { return !(fabsf(z) < INFINITY); };
  auto refuse = [&] {
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      a.logp[row] = __int_as_float(0x7fffffff);
    }
    sync();
  };
  if (!fine || bad(top)) {  // the same for every CTA of the cluster
    refuse();
    return;
  }
  const double per_logit = 1.4426950408889634074 / temp;
  Exp exp_of = {moved(ref), per_logit * 0x1p896, sh.tab};
  const float cf = (float)fmin(per_logit, 1e37);
  float zfloor = ref - 750.f * (float)temp;  // below it every e is zero: such logits are left out of counts, too
  auto refer_to = [&](float z) {
    ref = z;
    exp_of.ref = moved(z);
    zfloor = z - 750.f * (float)temp;
  };
  // After a walk that found `top`: whether the exponents were too far above their reference. (f64: 2^900; f32: 2^60)
  auto too_far = [&](float most) { return ((double)top - (double)ref) * per_logit > (double)most; };

  // ---- sums over the cluster, in rank order: N numbers per thread; every thread gets them
  int turn = 0;
  auto sums = [&](auto& v) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = warp_add(v[i]);
      if (lane == 0) sh.warp[warp][i] = v[i];
    }
    __syncthreads();
    if (tid < N) {
      double s = 0.0;
      for (int w = 0; w < kWarps; w++) s += sh.warp[w][tid];
      sh.x[turn][tid] = s;
    }
    sync();
#pragma unroll
    for (int i = 0; i < N; i++) {
      v[i] = 0.0;
      for (int q = 0; q < ranks; q++) v[i] += *of_rank(&sh.x[turn][i], q);
    }
    turn ^= 1;
  };

  // ---- what stays: z > tz, and z = tz up to index tidx
  float tz = -INFINITY;
  uint32_t tidx = 0xffffffffu;
  bool bounded = false;  // whether any is known
  auto stays = [&](float z, uint32_t i) { return z > tz || (z == tz && i <= tidx); };

  auto push = [&](float z, uint32_t i) {  // to rank 0's list: (~key, index), which sorts by falling z, then index
    const int n = atomicAdd(of_rank(&sh.count, 0), 1);
    if (n < kList) of_rank(list, 0)[n] = (unsigned long long)(~key_of(z)) << 32 | i;
  };
  auto sort_list = [&](int n) __attribute__((always_inline)) {  // by the threads of rank 0; up to the next power of two with ~0
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kThreads) list[i] = ~0ull;
    __syncthreads();
    for (int w = 2; w <= size; w *= 2)
      for (int s = w / 2; s; s /= 2) {
        for (int i = tid; i < size / 2; i += kThreads) {
          const int lo = 2 * i - (i & (s - 1)), hi = lo + s;
          const unsigned long long x = list[lo], y = list[hi];
          if ((x > y) == ((lo & w) == 0)) {
            list[lo] = y;
            list[hi] = x;
          }
        }
        __syncthreads();
      }
  };
  // Sums of what comes before in the list's order, thread t's eight entries from 8 t; `total` of all.
  auto list_scan = [&](const double (&e)[8], double& total) {
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < 8; j++) s += e[j];
    double inc = s;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sh.warp[warp][0] = inc;
    __syncthreads();
    double base = 0.0;
    total = 0.0;
    for (int w = 0; w < kWarps; w++) {
      if (w == warp) base = total;
      total += sh.warp[w][0];
    }
    __syncthreads();
    const double up = __shfl_up_sync(0xffffffffu, inc, 1);
    return base + (lane ? up : 0.0);
  };

  // ---- step 1: bins of d = ref - z by f32 weights among what stays so far; an interval [d0, d1] around the border. By
  // mass: equal steps of 3/8 T, from 6 T above the reference on; by count: quarters of octaves up to 750 T (beyond it e is zero).
  struct Span {
    float d0, d1;        // the border's interval
    double until, most;  // how much there is down to d1; the most tokens that the interval (all: everything down to d1) holds
    bool inside;         // it touches neither the first nor the last bin
  };
  auto bins = [&](auto walk, auto weighing, bool by_octave, bool all, double want, double fuzz, bool share, float lo,
                  float inv, bool fine_fuzz = false) __attribute__((always_inline)) {
    constexpr bool by_mass = decltype(weighing)::value;
    const int octaves = (int)(__float_as_uint(fmaxf(750.f * (float)temp, 1e-30f)) >> 21) - (kBins - 1);
    for (int b = 0; b < kBins; b++) hist[b * kThreads + tid] = 0.f;
    const float shift_b = -lo * inv;
    walk([&](const float(&z)[VEC], uint32_t i) {
      int b[VEC];
      float w[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float d = ref - z[j];
        if (by_octave) b[j] = min(max((int)(__float_as_uint(fmaxf(d, 0.f)) >> 21) - octaves, 0), kBins - 1);
        else  // rounded to the nearest bin by the sum with 1.5 * 2^23; -inf is in the last one and weighs nothing
          b[j] = __float_as_int(fminf(fmaxf(__fmaf_rn(d, inv, shift_b), 0.f), (float)(kBins - 1)) + 12582912.f) & (kBins - 1);
        if constexpr (by_mass) w[j] = exp2_fast(-d * cf);
        else w[j] = z[j] >= zfloor ? 1.f : 0.f;
        if (bounded) w[j] = stays(z[j], i + j) ? w[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; j++) hist[b[j] * kThreads + tid] += w[j];
    });
    __syncthreads();
    for (int b = warp; b < kBins; b += kWarps) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < kThreads / 32; q++) s += hist[b * kThreads + q * 32 + lane];
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) sh.x[turn][b] = (double)s;
    }
    sync();
    double bin[2];  // this lane's two bins, over the cluster; every warp alike
#pragma unroll
    for (int h = 0; h < 2; h++) {
      bin[h] = 0.0;
      for (int q = 0; q < ranks; q++) bin[h] += *of_rank(&sh.x[turn][2 * lane + h], q);
    }
    turn ^= 1;
    double inc = bin[0] + bin[1];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const double total = __shfl_sync(0xffffffffu, inc, 31);
    const double target = share ? want * total : want;
    // the first bin by whose end the border can have come, and the first by whose end it must have. The weights are off by a
    // share of what they are, so what lies behind the border is compared where that is less than what lies in front of it.
    const bool behind = fine_fuzz && total - target < target;
    double sum0 = inc - bin[1], sum1 = inc, goal = target, off = (fine_fuzz ? target : total) * fuzz;
    if (behind) {
      double suf = bin[0] + bin[1];
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const double down = __shfl_down_sync(0xffffffffu, suf, o);
        if (lane + o < 32) suf += down;
      }
      const double rest = (1.0 - want) * total;
      sum1 = -(suf - bin[0] - bin[1]);  // behind this lane's second bin
      sum0 = sum1 - bin[1];
      goal = -rest;
      off = rest * fuzz;
    }
    auto first_from = [&](double x) {
      const unsigned m0 = __ballot_sync(0xffffffffu, sum0 >= x), m1 = __ballot_sync(0xffffffffu, sum1 >= x);
      return min(m0 ? 2 * (__ffs(m0) - 1) : kBins - 1, m1 ? 2 * (__ffs(m1) - 1) + 1 : kBins - 1);
    };
    const int b0 = first_from(goal - off), b1 = first_from(goal + off);
    double members = 0.0, until = 0.0;
#pragma unroll
    for (int h = 0; h < 2; h++)
      if (2 * lane + h <= b1) {
        until += bin[h];
        if (2 * lane + h >= b0) members += bin[h];
      }
    members = warp_add(members);
    until = warp_add(until);
    __syncthreads();  // the bins may be cleared again
    Span r;
    r.until = until;
    r.inside = b0 > 0 && b1 < kBins - 1;
    if (by_octave) {
      r.d0 = b0 > 0 ? __uint_as_float((uint32_t)(b0 + octaves) << 21) : -INFINITY;
      r.d1 = b1 < kBins - 1 ? __uint_as_float((uint32_t)(b1 + 1 + octaves) << 21) : INFINITY;
    } else {
      const float step = 1.f / inv;
      r.d0 = b0 > 0 ? lo + ((float)b0 - 0.51f) * step : -INFINITY;
      r.d1 = b1 < kBins - 1 ? lo + ((float)b1 + 0.51f) * step : INFINITY;
    }
    // by mass, tokens are counted by the weight of the interval's far end
    r.most = all ? until : by_mass ? members * exp2((double)fmaxf(fminf(r.d1 * cf, 1000.f), -1000.f)) : members;
    return r;
  };
  const float mass_lo = -6.f * (float)temp, mass_inv = fminf((float)kBins / fmaxf(24.f * (float)temp, 1e-36f), 1e30f);
  auto walk_all = [&](auto f) { walk_part(Two(), warp, 0, its, f, nothing); };
  auto ends = [&](const Span& r, float& za, float& zb) {  // of logits, a little outside the interval's of d
    za = r.d0 > -INFINITY ? ref - (r.d0 - fabsf(r.d0) * 1e-6f) : INFINITY;
    zb = fmaxf(ref - (r.d1 + fabsf(r.d1) * 1e-6f), zfloor);
  };
  // By walks over all logits: the second and third one's 62 steps cut up the interval that the one before it showed.
  auto propose = [&](auto weighing, double want, bool share, bool all, float& za, float& zb) __attribute__((always_inline)) {
    constexpr bool by_mass = decltype(weighing)::value;
    const double fuzz = by_mass ? 3e-5 : 0.0;
    // (from the largest logit to 42 T below it, where e is 1e-18 of the largest)
    Span r = bins(walk_all, weighing, !by_mass, all, want, fuzz, share, 0.f, mass_inv * (24.f / 42.f), by_mass);
    for (int level = 1; level < 3; level++) {
      const float d0 = fmaxf(r.d0, 0.f);
      if (r.most <= 0.6 * kList || r.d1 == INFINITY || !(r.d1 > d0)) break;
      const float inv = fminf((float)(kBins - 2) / (r.d1 - d0), 1e30f), was0 = r.d0, was1 = r.d1;
      r = bins(walk_all, weighing, false, all, want, fuzz, share, d0 - 1.f / inv, inv, by_mass);
      r.d0 = fmaxf(r.d0, was0);  // the outer bins hold what is outside as well: there the ends stay
      r.d1 = fminf(r.d1, was1);
    }
    ends(r, za, zb);
  };

  // The border's key by bits, among the logits in [zb, za] whose order is not known; `above`: what the others above them weigh.
  auto search = [&](bool by_mass, double above, double want, float za, float zb) __attribute__((always_inline)) {
    auto in = [&](float z, uint32_t i) { return z <= za && z >= zb && stays(z, i); };
    auto weight_from = [&](uint32_t from) {
      double s[1] = {0.0};
      walk_part(One(), warp, 0, its,
                [&](const float(&z)[VEC], uint32_t i) {
#pragma unroll
                  for (int j = 0; j < VEC; j++)
                    if (in(z[j], i + j) && key_of(z[j]) >= from) s[0] += by_mass ? exp_of(z[j]) : 1.0;
                },
                nothing);
      sums(s);
      return s[0];
    };
    float low = INFINITY, high = -INFINITY;
    walk_part(One(), warp, 0, its,
              [&](const float(&z)[VEC], uint32_t i) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                  if (in(z[j], i + j)) low = fminf(low, z[j]), high = fmaxf(high, z[j]);
              },
              nothing);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    __syncthreads();
    if (lane == 0) {
      sh.fwarp[warp][2] = low;
      sh.fwarp[warp][3] = high;
    }
    sync();
    for (int q = 0; q < ranks; q++) {
      const float* other = of_rank(&sh.fwarp[0][0], q);
      for (int w = 0; w < kWarps; w++) {
        low = fminf(low, other[4 * w + 2]);
        high = fmaxf(high, other[4 * w + 3]);
      }
    }
    const uint32_t klow = key_of(low), khigh = key_of(high);
    const int bits = klow == khigh ? 0 : 32 - __clz(klow ^ khigh);
    want = fmin(want, above + weight_from(0));
    uint32_t key = bits == 32 ? 0u : khigh >> bits << bits;  // what the members' keys have in common
    for (int b = bits - 1; b >= 0; b--)
      if (above + weight_from(key | 1u << b) >= want) key |= 1u << b;
    if (key != 0xffffffffu) above += weight_from(key + 1);
    // so many of its equals as are needed, the lowest indices first
    const float z0 = of_key(key);
    double equals[1] = {0.0};
    walk_part(One(), warp, 0, its,
              [&](const float(&z)[VEC], uint32_t i) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                  if (z[j] == z0 && stays(z[j], i + j)) equals[0] += 1.0;
              },
              nothing);
    const double own = warp_add(equals[0]);
    sums(equals);
    double before = 0.0;
    for (int q = 0; q < rank; q++) before += *of_rank(&sh.x[turn ^ 1][0], q);
    const double e0 = by_mass ? exp_of(z0) : 1.0;
    double need = fmin(fmax(ceil((want - above) / e0), 1.0), equals[0]);
    if (need > 1.0 && above + (need - 1.0) * e0 >= want) need -= 1.0;  // the quotient's rounding
    if (tid == 0) sh.found = -1;
    if (lane == 0) sh.warp[warp][0] = own;
    __syncthreads();
    for (int w = 0; w < warp; w++) before += sh.warp[w][0];
    if (before < need && need <= before + own) {  // the warp that holds the need-th equal
      walk_part(One(), warp, 0, its,
                [&](const float(&z)[VEC], uint32_t i) {
                  int n = 0;
#pragma unroll
                  for (int j = 0; j < VEC; j++) n += z[j] == z0 && stays(z[j], i + j);
                  int inc = n;
                  for (int o = 1; o < 32; o *= 2) {
                    const int up = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += up;
                  }
                  int left = (int)(need - before) - (inc - n);  // this lane's left-th is the one
                  if (left >= 1 && left <= n) {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                      if (z[j] == z0 && stays(z[j], i + j) && --left == 0) sh.found = (int)i + j;
                  }
                  before += (double)__shfl_sync(0xffffffffu, inc, 31);
                },
                nothing);
    }
    sync();
    int found = -1;
    for (int q = 0; q < ranks; q++) found = max(found, *of_rank(&sh.found, q));
    sync();
    tz = z0;
    tidx = (uint32_t)found;
    bounded = true;
  };
  // The border in rank 0's list of n: the last entry before which less than `want` comes, `above` included.
  auto border = [&](bool by_mass, double above, double want, int n) __attribute__((always_inline)) {
    int m = 0;
    if (rank == 0) {
      sort_list(n);
      double e[8], total;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int i = 8 * tid + j;
        e[j] = i < n ? (by_mass ? exp_of(of_key(~(uint32_t)(list[i] >> 32))) : 1.0) : 0.0;
      }
      double at = above + list_scan(e, total);
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (8 * tid + j < n && at < want) mine = 8 * tid + j;
        at += e[j];
      }
      mine = __reduce_max_sync(0xffffffffu, mine);
      if (lane == 0) sh.iwarp[warp] = mine;
      __syncthreads();
      if (tid == 0) {
        for (int w = 0; w < kWarps; w++) mine = max(mine, sh.iwarp[w]);
        sh.tz = of_key(~(uint32_t)(list[mine] >> 32));
        sh.tidx = (uint32_t)list[mine];
        sh.found = mine + 1;
      }
    }
    sync();
    tz = *of_rank(&sh.tz, 0);
    tidx = *of_rank(&sh.tidx, 0);
    bounded = true;
    m = *of_rank(&sh.found, 0);
    sync();
    return m;
  };

  // The listing of what is in [zb, za], by count; `above` it
  auto list_walk = [&](float za, float zb, bool all, double& above, float& most) {
    double n[1] = {0.0};
    float m = -INFINITY;
    walk_part(Four(), warp, 0, its,
              [&](const float(&z)[VEC], uint32_t i) {
                const float high = largest(z, -INFINITY);
                m = max_nan(m, high);
                if (high < zb) return;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                  if (!(z[j] >= zb)) continue;
                  if (z[j] > za && !all) n[0] += 1.0;
                  else push(z[j], i + j);
                }
              },
              nothing);
    most = max_of_all(m);
    sums(n);
    above = n[0];
    const int listed = *of_rank(&sh.count, 0);
    sync();
    if (tid == 0) sh.count = 0;
    return listed;
  };
  if (k > 0) {
    float za = INFINITY, zb = zfloor;
    double above = 0.0;
    int n = kList + 1;
    if (few) {
      // the sample's share of k, and four of its standard deviations and a few more: a list of all that is above that
      const double share = fmin(1.0, (double)(kSample * kThreads) * VEC * ranks / a.V);
      const double of_k = share * k, want = share < 1.0 ? of_k + 4.0 * sqrt(of_k) + 8.0 : (double)k;
      const Span r = bins(walk_sample, ByCount(), true, true, want, 0.0, false, 0.f, 0.f);
      float most = top;
      if (r.until <= 0.8 * share * kList || r.until < want) {  // (less than wanted: the sample has no more that count)
        if (r.until >= want) ends(r, za, zb);
        n = list_walk(INFINITY, zb, true, above, most);
        known = true;
        top = most;
      }
    }
    if (!known) walk_max(), known = true;
    if (bad(top)) {
      refuse();
      return;
    }
    if (ref != top) {
      // what is left out below zfloor has no mass beside the largest either
      const float was = zfloor;
      refer_to(top);
      if (zb == was) zb = zfloor;
    }
    if (!(few && n <= kList && (n >= k || zb == zfloor))) {
      propose(ByCount(), (double)k, false, few, za, zb);
      float unused;
      n = list_walk(za, zb, few, above, unused);
    }
    if (few && n <= kList && (n >= k || zb == zfloor)) {  // the list holds all of the first k: the rest is rank 0's
      if (rank == 0) {
        sort_list(n);
        const int m = n < k ? n : k;
        double e[8], total;
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = 8 * tid + j < m ? exp_of(of_key(~(uint32_t)(list[8 * tid + j] >> 32))) : 0.0;
        double at = list_scan(e, total);
        // top-p and min-p end the sorted list somewhere; what is left is sorted by index
        unsigned long long mine[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int i = 8 * tid + j;
          const bool in = i < m && (i == 0 || ((top_p >= 1.0 || at < top_p * total) && e[j] >= min_p));
          mine[j] = in ? (list[i] << 32) | (uint32_t)~(uint32_t)(list[i] >> 32) : ~0ull;  // (index, key)
          at += e[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (8 * tid + j < m) list[8 * tid + j] = mine[j];
        __syncthreads();
        sort_list(m);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          mine[j] = 8 * tid + j < m ? list[8 * tid + j] : ~0ull;
          e[j] = mine[j] == ~0ull ? 0.0 : exp_of(of_key((uint32_t)mine[j]));
        }
        at = list_scan(e, total);
        const double target = u * total;
        int pick = -1, back = -1;  // the first whose sum passes the target; the last with any mass
#pragma unroll
        for (int j = 0; j < 8; j++) {
          at += e[j];
          if (e[j] > 0.0) {
            back = 8 * tid + j;
            if (pick < 0 && at > target) pick = back;
          }
        }
        const unsigned lowest = __reduce_min_sync(0xffffffffu, (unsigned)pick);
        back = __reduce_max_sync(0xffffffffu, back);
        if (lane == 0) {
          sh.iwarp[warp] = (int)lowest;
          sh.fwarp[warp][0] = __int_as_float(back);
        }
        __syncthreads();
        if (tid == 0) {
          unsigned best = 0xffffffffu;
          for (int w = 0; w < kWarps; w++) {
            best = min(best, (unsigned)sh.iwarp[w]);
            back = max(back, __float_as_int(sh.fwarp[w][0]));
          }
          const unsigned long long e1 = list[best != 0xffffffffu ? (int)best : max(back, 0)];
          a.token[row] = (int)(e1 >> 32);
          a.logp[row] = (float)(((double)of_key((uint32_t)e1) - (double)ref) / temp - log(total));
        }
      }
      sync();
      return;
    }
    if (!few && n <= kList && above < (double)k && above + n >= (double)k)
      border(false, above, (double)k, n);
    else if (few || zb > zfloor || above + n >= (double)k)  // (otherwise no more than k have any mass)
      search(false, 0.0, (double)k, INFINITY, zfloor);
  }

  // ---- step 2: the f64 walk. Above [zb, za] what stays goes into sums by warp, segment of its iterations, and lane; the
  // members, and all of it, into sums of their own.
  const int seg_its = (its + kSegs - 1) / kSegs;
  double w3[3];  // mass above, in, and of all
  constexpr int kPlain = 0, kKept = 1, kListing = 2;
  auto f64_walk = [&](auto mode, float za, float zb, double floor) {
    constexpr int MODE = decltype(mode)::value;
    double s = 0.0;
    float m = -INFINITY;
    w3[0] = w3[1] = w3[2] = 0.0;
    for (int g = 0; g < kSegs; g++) sub[(warp * kSegs + g) * 32 + lane] = 0.0;
    walk_part(Two(), warp, 0, its,
              [&](const float(&z)[VEC], uint32_t i) {
                double e[VEC];
#pragma unroll
                for (int j = 0; j < VEC; j += 4) exp_of.template many<4>(z + j, e + j);
                if constexpr (MODE == kPlain) {
                  m = largest(z, m);
#pragma unroll
                  for (int j = 0; j < VEC; j++) s += e[j];
                } else if constexpr (MODE == kKept) {
#pragma unroll
                  for (int j = 0; j < VEC; j++) s += stays(z[j], i + j) && e[j] >= floor ? e[j] : 0.0;
                } else {
                  unsigned in = 0;
#pragma unroll
                  for (int j = 0; j < VEC; j++) {
                    if (bounded) e[j] = stays(z[j], i + j) ? e[j] : 0.0;
                    w3[2] += e[j];
                    s += z[j] > za ? e[j] : 0.0;
                    if (z[j] <= za && z[j] >= zb) in |= 1u << j;
                  }
                  if (in) {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                      if ((in >> j & 1) && e[j] > 0.0) {
                        w3[1] += e[j];
                        push(z[j], i + j);
                      }
                  }
                }
              },
              [&](int it) {
                if ((it + 1) % seg_its == 0 || it + 1 == its) {
                  sub[(warp * kSegs + it / seg_its) * 32 + lane] = s;
                  w3[0] += s;
                  s = 0.0;
                }
              });
    return m;
  };
  using Plain = std::integral_constant<int, kPlain>;
  using Kept = std::integral_constant<int, kKept>;
  using Listing = std::integral_constant<int, kListing>;
  bool summed = false;
  int members = 0;  // of rank 0's list that stay, in `sub` not counted
  if (plain) {
    for (;;) {
      const float m = max_of_all(f64_walk(Plain(), 0.f, 0.f, 0.0));
      top = m;
      if (bad(top)) {
        refuse();
        return;
      }
      if (!too_far(900.f)) break;
      refer_to(top);
    }
    summed = true;
  }
  if (top_p < 1.0) {
    float za, zb;
    bool proposed = false;
    if (!known) {
      // the sample's interval, with 6 % of the mass on either side for its error, cut up by one walk over all
      const Span r = bins(walk_sample, ByMass(), false, false, top_p, 0.06, true, mass_lo, mass_inv);
      const float d0 = fmaxf(r.d0, mass_lo), d1 = fminf(r.d1, mass_lo + (float)kBins / mass_inv);
      const float inv = fminf((float)(kBins - 2) / (d1 - d0), 1e30f);
      float m = -INFINITY;
      const Span all = bins(
          [&](auto f) {
            walk_part(Two(), warp, 0, its,
                      [&](const float(&z)[VEC], uint32_t i) {
                        m = largest(z, m);
                        f(z, i);
                      },
                      nothing);
          },
          ByMass(), false, false, top_p, 3e-5, true, d0 - 1.f / inv, inv, true);
      top = max_of_all(m);
      known = true;
      if (bad(top)) {
        refuse();
        return;
      }
      if (all.inside && all.most <= 0.6 * kList && !too_far(60.f)) {
        ends(all, za, zb);
        proposed = true;
      }
    }
    if (!proposed) {
      refer_to(top);
      propose(ByMass(), top_p, true, false, za, zb);
    }
    f64_walk(Listing(), za, zb, 0.0);
    sums(w3);
    const int n = *of_rank(&sh.count, 0);
    sync();
    if (tid == 0) sh.count = 0;
    const double want = top_p * w3[2];
    const bool inside = w3[0] < want && w3[0] + w3[1] >= want;
    if (inside && n <= kList) {
      members = border(true, w3[0], want, n);
      summed = min_p <= 0.0;
    } else if (inside) {
      search(true, w3[0], want, za, zb);
    } else {
      search(true, 0.0, want, INFINITY, zfloor);
    }
  }

  // ---- the draw: the segment that holds u's place is walked once more
  const double floor = min_p > 0.0 ? min_p * exp_of(top) : 0.0;
  if (!summed) {
    __syncthreads();
    f64_walk(Kept(), 0.f, 0.f, floor);
    members = 0;
  }
  __syncthreads();
  if (members) {  // the listed ones' masses and segments
    const unsigned long long* from = of_rank(list, 0);
    for (int j = tid; j < members; j += kThreads) {
      const uint32_t i = (uint32_t)from[j];
      const bool mine = i >= (uint32_t)first && i < (uint32_t)last;
      const int v = ((int)(i - (uint32_t)first) + shift) / VEC;
      sh.part[j] = (unsigned char)(mine ? v / per_warp * kSegs + v % per_warp / 32 / seg_its : 255);
      list_e[j] = mine ? exp_of(of_key(~(uint32_t)(from[j] >> 32))) : 0.0;
    }
    __syncthreads();
  }
  if (tid < kWarps * kSegs) {
    double s = 0.0;
    for (int l = 0; l < 32; l++) s += sub[tid * 32 + ((l + tid) & 31)];
    for (int j = 0; j < members; j++)
      if (sh.part[j] == tid) s += list_e[j];
    sh.seg[tid] = s;
  }
  __syncthreads();
  // u's place is in the last rank, and there in the last segment, that has any mass and does not begin behind it; where
  // rounding (or u = 1) leaves the target unreached there, its last token with any mass is the one
  double part[4], inc = 0.0;
#pragma unroll
  for (int j = 0; j < 4; j++) inc += part[j] = sh.seg[4 * lane + j];
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const double up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (tid == 31) sh.x[turn][0] = inc;
  sync();
  int holder = -1;
  double before = 0.0, total = 0.0;
  for (int q = 0; q < ranks; q++) total += *of_rank(&sh.x[turn][0], q);
  const double target = u * total;
  double from = 0.0;
  for (int q = 0; q < ranks; q++) {
    const double x = *of_rank(&sh.x[turn][0], q);
    if (x > 0.0 && from <= target) holder = q, before = from;
    from += x;
  }
  if (holder < 0) {  // no mass anywhere, though the largest logit's e is at least 1: an answer all the same
    refuse();
    return;
  }
  if (rank == holder && warp == 0) {
    const double up = __shfl_up_sync(0xffffffffu, inc, 1);
    double at = before + (lane ? up : 0.0), start = before;
    int held = -1;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (part[j] > 0.0 && at <= target) held = 4 * lane + j, start = at;
      at += part[j];
    }
    const int seg = __reduce_max_sync(0xffffffffu, held);
    at = __shfl_sync(0xffffffffu, start, seg / 4);
    const int w = seg / kSegs, i0 = seg % kSegs * seg_its, i1 = min(its, i0 + seg_its);
    int pick = -1, back = -1;
    walk_part(One(), w, i0, i1,
              [&](const float(&z)[VEC], uint32_t i) {
                double e[VEC], mine = 0.0;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                  e[j] = exp_of(z[j]);
                  e[j] = stays(z[j], i + j) && e[j] >= floor ? e[j] : 0.0;
                  mine += e[j];
                }
                double inc = mine;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                  const double up = __shfl_up_sync(0xffffffffu, inc, o);
                  if (lane >= o) inc += up;
                }
                const double up = __shfl_up_sync(0xffffffffu, inc, 1);
                double here = at + (lane ? up : 0.0);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                  here += e[j];
                  if (e[j] > 0.0) {
                    back = (int)i + j;
                    if (pick < 0 && here > target) pick = back;
                  }
                }
                at += __shfl_sync(0xffffffffu, inc, 31);
              },
              nothing);
    const unsigned lowest = __reduce_min_sync(0xffffffffu, (unsigned)pick);
    back = __reduce_max_sync(0xffffffffu, back);
    const int token = lowest != 0xffffffffu ? (int)lowest : back;
    if (lane == 0) {
      float z;
      if constexpr (VEC == 4) z = src[token - first];
      else z = __bfloat162float(src[token - first]);
      a.token[row] = token;
      a.logp[row] = (float)(((double)z - (double)ref) / temp - log(total));
    }
  }
  sync();
}

template <typename T, bool SOLO>
static int sample_variant(const SampleArgs& a, long rows, int ranks, cudaStream_t st) {
  const size_t smem = sizeof(float) * kBins * kThreads + (SOLO ? 0 : (size_t)a.slice * sizeof(T) + 32);
  int rc = raise_smem((const void*)sample_kernel<T, SOLO>, smem);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(rows * ranks);
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = SOLO ? 1 : 2;
  PL_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T, SOLO>, a));
  count_launch();
  return PL_OK;
}
template <typename T>
static int sample_launch(SampleArgs& a, long rows, cudaStream_t st) {
  // Few rows are split over clusters of four, in parts of 4,096 values and more, as long as the clusters fit on the device at once
  // (66 of four at two CTAs per SM; more run when the first are done). us whole / in four:
  //              bf16 rows of 8,192   16,384     32,768     65,536     131,072     f32 of 32,768   65,536
  //   top_k 50,  32 rows  18 / 22     22 / 23    25 / 24    31 / 28    45 / 33     32 / 25         39 / 30
  //              64       17 / 25     22 / 25    25 / 26    32 / 31    58 / 60     27 / 28         41 / 55
  //              100      18 / 44     22 / 46    25 / 48    37 / 55    48 / 106    32 / 51         39 / 101
  //   top_p,     32       35 / 38     64 / 46    69 / 49    115 / 60   202 / 85    74 / 62         124 / 65
  //              64       39 / 45     51 / 53    69 / 60    113 / 77   202 / 153   75 / 64         124 / 110
  //              100      39 / 76     55 / 79    81 / 93    114 / 120  202 / 225   78 / 91         124 / 164
  // Clusters of two gained up to a tenth between 75 and 148 rows of 32,768 and lost as much and more elsewhere. A part has to fit
  // into shared memory: rows of more than 384 KB go in eight (131,072 f32, top_p, 32 rows 234 / 150, 64 226 / 267).
  const int parts = (long)a.V * sizeof(T) > 4 * 98304L ? 8 : 4;
  const int ranks = a.V >= 16384 && rows * parts <= 264 ? parts : 1;
  a.slice = (int)round_up(ceil_div(a.V, ranks), 8);
  return ranks == 1 ? sample_variant<T, true>(a, rows, 1, st) : sample_variant<T, false>(a, rows, ranks, st);
}

}  // namespace pl

extern "C" int pl_sample_dev(const void* logits, size_t ld, size_t rows, size_t V, uint8_t bf16, const float* u,
                             const float* temperature, double temperature_all, const int32_t* top_k, size_t top_k_all,
                             const float* top_p, double top_p_all, const float* min_p, double min_p_all, int32_t* token,
                             float* logp, void* stream) {
  using namespace pl;
  const char* me = "pl_sample_dev";
  PL_REQUIRE(V > 0 && V <= (size_t)kMostVocab, PL_ERR_INVALID, "%s: %zu tokens, 1 to %d wanted", me, V, kMostVocab);
  PL_REQUIRE(ld >= V, PL_ERR_INVALID, "%s: a row stride of %zu, below %zu tokens", me, ld, V);
  PL_REQUIRE(rows <= (1u << 27), PL_ERR_INVALID, "%s: %zu rows are too many", me, rows);
  PL_REQUIRE(temperature || (temperature_all >= 0.0 && temperature_all < INFINITY), PL_ERR_INVALID, "%s: temperature = %g", me,
             temperature_all);
  PL_REQUIRE(top_p || top_p_all == top_p_all, PL_ERR_INVALID, "%s: top_p = %g", me, top_p_all);
  PL_REQUIRE(min_p || min_p_all == min_p_all, PL_ERR_INVALID, "%s: min_p = %g", me, min_p_all);
  if (rows == 0) return PL_OK;
  PL_REQUIRE(logits && u && token && logp, PL_ERR_INVALID, "%s: NULL logits, numbers or results", me);
  PL_REQUIRE((uintptr_t)logits % (bf16 ? 2 : 4) == 0, PL_ERR_INVALID, "%s: logits are not aligned to their type", me);
  int rc = require_device();
  if (rc) return rc;
  SampleArgs a = {logits, (long)ld, (int)V, 0, u, temperature, top_p, min_p, (const int*)top_k, temperature_all, top_p_all,
                  min_p_all, (int)(top_k_all < V ? top_k_all : 0), token, logp};
  return bf16 ? sample_launch<__nv_bfloat16>(a, (long)rows, (cudaStream_t)stream)
              : sample_launch<float>(a, (long)rows, (cudaStream_t)stream);
}
