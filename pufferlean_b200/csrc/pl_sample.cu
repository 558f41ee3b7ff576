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
// Many rows: a CTA per row, which walks it again for each step below (from L2: the rows in flight fit there). Few rows: a cluster of
// CTAs per row, each with a contiguous slice in shared memory.
//
// The border of top-k or top-p is found in three steps. (1) One or two walks with f32 weights put counts or masses into 64
// bins of d = max - z, each thread's its own (no atomics), the second walk's around the border that the first one shows:
// this proposes an interval [zb, za] of logits. (2) A walk in f64 takes the masses above, in and below the interval and
// lists what lies in it. (3) If these say that the border is inside, which they do but for a few rows in a million, the list is
// sorted and the border is exact. Otherwise, or if the list overflows (more equal logits than it holds), the border's
// key is searched bit by bit. So the f32 sums cost time where they are off, never a token.
//
// Bound by the f64 pipe: one walk of 11 f64 operations per logit is 5.5 clocks per 32 logits on an SM, 100 us at 1,024 x
// 131,072 (HBM: 41 us in bf16).
#include <cooperative_groups.h>

#include <type_traits>

#include "pl_common.cuh"
#include "pl_runtime.h"

namespace cg = cooperative_groups;

namespace pl {

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 64, kList = 2048, kSegs = 16;
constexpr int kMostVocab = 1 << 18;

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

// exp((z - max) / T) in f64: 2^y, y = n / 16 + r with 2^(n / 16) from a table and 2^r, |r| <= 1/32, from five terms of its series
// (the sixth is 1.4e-13 of the value at most).
struct Exp {
  double max, c;  // c = log2(e) / T
  const double* tab;
  __device__ __forceinline__ double operator()(float z) const {
    // the f32's bits as a double (a conversion has a quarter of the rate); below 2^-126 it is off by as little
    const uint32_t b = __float_as_uint(z);
    const double d = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + (896u << 20))), (int)(b << 29));
    const double y = (d - max) * c;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
    const double s = fma(y, 16.0, magic);
    const int n = __double2loint(s);
    const double r = fma(s - magic, -0.0625, y);
    const double l = 0.6931471805599453094;
    double q = l * l * l * l * l / 120.0;
    q = fma(q, r, l * l * l * l / 24.0);
    q = fma(q, r, l * l * l / 6.0);
    q = fma(q, r, l * l / 2.0);
    q = fma(q, r, l);
    q = fma(q, r, 1.0) * tab[n & 15];
    const double e = __hiloint2double(__double2hiint(q) + (n >> 4) * (1 << 20), __double2loint(q));
    return (uint32_t)__double2hiint(y) < 0xc08f4000u ? e : 0.0;  // y > -1000: by the order of negative doubles' bits
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
  double temp = fmin(t_given, 1e30), top_p = p_given, min_p = fmin(mp_given, 1.0);
  const double u = fmin(fmax(u_given, 0.0), 1.0);
  const bool fine = t_given >= 0.0 && t_given < INFINITY && p_given == p_given && mp_given == mp_given && u_given == u_given;
  if (temp == 0.0 || top_p <= 0.0) k = 1;  // the first in order alone
  if (k == 1) {
    temp = 1.0;
    top_p = 1.0;
    min_p = 0.0;
  }
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
  // f(value, index in the row) for the values of warp w's iterations [i0, i1), and done(iteration) behind each; U vectors are
  // loaded at a time.
  auto walk_part = [&](auto unroll, int w, int i0, int i1, auto f, auto done) {
    constexpr int U = decltype(unroll)::value;
    for (int it = i0; it < i1; it += U) {
      uint4 x[U];
#pragma unroll
      for (int q = 0; q < U; q++) {
        const int v = w * per_warp + (it + q) * 32 + lane;
        if (it + q < i1 && v < vecs) {
          if constexpr (SOLO) x[q] = fetch(v);
          else x[q] = *reinterpret_cast<const uint4*>(cache + v * VEC);
        } else {
          const uint32_t none = VEC == 4 ? 0xff800000u : 0xff80ff80u;
          x[q] = make_uint4(none, none, none, none);
        }
      }
#pragma unroll
      for (int q = 0; q < U; q++) {
        const uint32_t i = (uint32_t)(first + (w * per_warp + (it + q) * 32 + lane) * VEC - shift);
#pragma unroll
        for (int j = 0; j < VEC; j++) f(value(x[q], j), i + j);
        if (it + q < i1) done(it + q);
      }
    }
  };
  auto nothing = [](int) {};
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;

  // ---- the largest logit
  float top = -INFINITY, nan = 0.f;
  if constexpr (!SOLO) {
    for (int it = 0; it < its; it++) {
      const int v = warp * per_warp + it * 32 + lane;
      if (v < vecs) *reinterpret_cast<uint4*>(cache + v * VEC) = fetch(v);
    }  // a thread reads what it stored itself
  }
  walk_part(Four(), warp, 0, its,
            [&](float z, uint32_t) {
              top = fmaxf(top, z);
              if (z != z) nan = 1.f;
            },
            nothing);
  if (tid < 16) sh.tab[tid] = exp2((double)tid / 16.0);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    nan = fmaxf(nan, __shfl_xor_sync(0xffffffffu, nan, o));
  }
  if (lane == 0) {
    sh.fwarp[warp][0] = top;
    sh.fwarp[warp][1] = nan;
  }
  if (tid == 0) sh.count = 0;
  sync();
  top = -INFINITY, nan = 0.f;
  for (int q = 0; q < ranks; q++) {
    const float* other = of_rank(&sh.fwarp[0][0], q);
    for (int w = 0; w < kWarps; w++) {
      top = fmaxf(top, other[4 * w]);
      nan = fmaxf(nan, other[4 * w + 1]);
    }
  }
  if (!fine || nan != 0.f || fabsf(top) == INFINITY) {  // the same for every CTA of the cluster
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      a.logp[row] = __int_as_float(0x7fffffff);
    }
    sync();
    return;
  }
  const Exp exp_of = {(double)top, 1.4426950408889634074 / temp, sh.tab};
  const float cf = (float)fmin(exp_of.c, 1e37);

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
  auto stays = [&](float z, uint32_t i) { return z > tz || (z == tz && i <= tidx); };

  auto push = [&](float z, uint32_t i) {  // to rank 0's list: (~key, index), which sorts by falling z, then index
    const int n = atomicAdd(of_rank(&sh.count, 0), 1);
    if (n < kList) of_rank(list, 0)[n] = (unsigned long long)(~key_of(z)) << 32 | i;
  };
  auto sort_list = [&](int n) {  // by the threads of rank 0; up to the next power of two with ~0
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

  // Below it every e is zero: such logits are left out of counts, too.
  const float zfloor = top - 750.f * (float)temp;

  // ---- step 1: bins of d = (max - z) by f32 weights among what stays so far; [lo, hi] of d around the border. By mass: equal
  // steps of 3/8 T; by count: quarters of octaves up to 750 T (beyond it e is zero); then 62 steps of the interval.
  // Ends when about `room` members are left, or the weight of the interval and all above it (all) is.
  auto propose = [&](bool by_mass, double want, bool share, bool all, float& za, float& zb) {
    const float end = 750.f * (float)temp;
    float lo = 0.f, inv = (float)kBins / fmaxf(24.f * (float)temp, 1e-36f);
    const int octaves = (int)(__float_as_uint(fmaxf(end, 1e-30f)) >> 21) - (kBins - 1);
    float d0 = 0.f, d1 = INFINITY;
    for (int level = 0; level < 3; level++) {
      const bool by_octave = level == 0 && !by_mass;
      for (int b = 0; b < kBins; b++) hist[b * kThreads + tid] = 0.f;
      walk_part(Two(), warp, 0, its,
                [&](float z, uint32_t i) {
                  if (!(z >= zfloor) || !stays(z, i)) return;
                  const float d = top - z;
                  int b;
                  if (by_octave) b = min(max((int)(__float_as_uint(d) >> 21) - octaves, 0), kBins - 1);
                  else b = __float_as_int(fminf(fmaxf((d - lo) * inv, 0.f), (float)(kBins - 1)) + 12582912.f) & (kBins - 1);
                  hist[b * kThreads + tid] += by_mass ? exp2_fast(-d * cf) : 1.f;
                },
                nothing);
      __syncthreads();
      for (int b = warp; b < kBins; b += kWarps) {
        double s = 0.0;
        for (int q = 0; q < kThreads / 32; q++) s += (double)hist[b * kThreads + q * 32 + lane];
        s = warp_add(s);
        if (lane == 0) sh.x[turn][b] = s;
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
      const double target = share ? want * total : want, fuzz = by_mass ? 3e-5 * total : 0.0;
      // the first bin at whose end the border can have come, and the first by whose end it must have
      const double end0 = inc - bin[1], end1 = inc;
      const unsigned can0 = __ballot_sync(0xffffffffu, end0 >= target - fuzz), can1 = __ballot_sync(0xffffffffu, end1 >= target - fuzz);
      const unsigned must0 = __ballot_sync(0xffffffffu, end0 >= target + fuzz), must1 = __ballot_sync(0xffffffffu, end1 >= target + fuzz);
      auto first_of = [](unsigned m0, unsigned m1) {
        const int i0 = m0 ? 2 * (__ffs(m0) - 1) : kBins - 1, i1 = m1 ? 2 * (__ffs(m1) - 1) + 1 : kBins - 1;
        return min(i0, i1);
      };
      const int b0 = first_of(can0, can1), b1 = first_of(must0, must1);
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
      // bins 0 and 63 hold what is outside as well: there the interval's ends stay as they were
      if (by_octave) {
        if (b0 > 0) d0 = __uint_as_float((uint32_t)(b0 + octaves) << 21);
        if (b1 < kBins - 1) d1 = __uint_as_float((uint32_t)(b1 + 1 + octaves) << 21);
      } else {
        const float step = 1.f / inv;
        if (b0 > 0) d0 = fmaxf(d0, lo + ((float)b0 - 0.51f) * step);
        if (b1 < kBins - 1) d1 = fminf(d1, lo + ((float)b1 + 0.51f) * step);
      }
      za = d0 > 0.f ? top - d0 * 0.999999f : INFINITY;
      zb = fmaxf(top - d1 * 1.000001f, zfloor);
      // by mass, the bin's tokens are counted by the weight of its far end
      const double many = all ? until : by_mass ? members * exp2((double)fminf(d1 * cf, 1000.f)) : members;
      if (many <= 0.6 * kList || d1 == INFINITY || !(d1 > d0)) break;
      inv = fminf((float)(kBins - 2) / (d1 - d0), 1e30f);
      lo = d0 - 1.f / inv;
    }
  };

  // The border's key by bits, among the logits in [zb, za] whose order is not known; `above`: what the others above them weigh.
  auto search = [&](bool by_mass, double above, double want, float za, float zb) {
    auto in = [&](float z, uint32_t i) { return z <= za && z >= zb && stays(z, i); };
    auto weight_from = [&](uint32_t from) {
      double s[1] = {0.0};
      walk_part(One(), warp, 0, its,
                [&](float z, uint32_t i) {
                  if (in(z, i) && key_of(z) >= from) s[0] += by_mass ? exp_of(z) : 1.0;
                },
                nothing);
      sums(s);
      return s[0];
    };
    float low = INFINITY, high = -INFINITY;
    walk_part(One(), warp, 0, its,
              [&](float z, uint32_t i) {
                if (in(z, i)) low = fminf(low, z), high = fmaxf(high, z);
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
              [&](float z, uint32_t i) {
                if (z == z0 && stays(z, i)) equals[0] += 1.0;
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
      int n = 0;
      uint32_t mine[VEC];
      walk_part(One(), warp, 0, its,
                [&](float z, uint32_t i) {
                  const bool is = z == z0 && stays(z, i);
#pragma unroll
                  for (int j = 0; j < VEC; j++)
                    if (is && n == j) mine[j] = i;
                  n += is;
                },
                [&](int) {
                  int inc = n;
                  for (int o = 1; o < 32; o *= 2) {
                    const int up = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += up;
                  }
                  const int left = (int)(need - before) - (inc - n);  // this lane's left-th is the one
#pragma unroll
                  for (int j = 0; j < VEC; j++)
                    if (left == j + 1 && left <= n) sh.found = (int)mine[j];
                  before += (double)__shfl_sync(0xffffffffu, inc, 31);
                  n = 0;
                });
    }
    sync();
    int found = -1;
    for (int q = 0; q < ranks; q++) found = max(found, *of_rank(&sh.found, q));
    sync();
    tz = z0;
    tidx = (uint32_t)found;
  };
  // The border in rank 0's list of n: the last entry before which less than `want` comes, `above` included.
  auto border = [&](bool by_mass, double above, double want, int n) {
    int m = 0;
    if (rank == 0) {
      sort_list(n);
      double e[8], total;
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] = 8 * tid + j < n ? (by_mass ? exp_of(of_key(~(uint32_t)(list[8 * tid + j] >> 32))) : 1.0) : 0.0;
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
    m = *of_rank(&sh.found, 0);
    sync();
    return m;
  };

  if (k > 0) {
    float za, zb;
    const bool few = k <= kList / 2;
    propose(false, (double)k, false, few, za, zb);
    double above[1] = {0.0};
    walk_part(Four(), warp, 0, its,
              [&](float z, uint32_t i) {
                if (z > za && !few) above[0] += 1.0;
                else if (z >= zb) push(z, i);
              },
              nothing);
    sums(above);
    const int n = *of_rank(&sh.count, 0);
    sync();
    if (tid == 0) sh.count = 0;
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
          const unsigned long long e1 = list[best != 0xffffffffu ? (int)best : back];
          a.token[row] = (int)(e1 >> 32);
          a.logp[row] = (float)(((double)of_key((uint32_t)e1) - (double)top) / temp - log(total));
        }
      }
      sync();
      return;
    }
    if (!few && n <= kList && above[0] < (double)k && above[0] + n >= (double)k)
      border(false, above[0], (double)k, n);
    else if (few || zb > zfloor || above[0] + n >= (double)k)  // (otherwise no more than k have any mass)
      search(false, 0.0, (double)k, INFINITY, zfloor);
  }

  // ---- step 2: the f64 walk. Above [zb, za] what stays goes into sums by warp, segment of its iterations, and lane; the rest of it,
  // and the members, into sums of their own.
  const int seg_its = (its + kSegs - 1) / kSegs;
  double w3[3];  // mass above, in, below
  auto f64_walk = [&](float za, float zb, double floor, bool listing) {
    double s = 0.0;
    w3[0] = w3[1] = w3[2] = 0.0;
    for (int g = 0; g < kSegs; g++) sub[(warp * kSegs + g) * 32 + lane] = 0.0;
    walk_part(Two(), warp, 0, its,
              [&](float z, uint32_t i) {
                double e = exp_of(z);
                e = stays(z, i) && e >= floor ? e : 0.0;
                if (!listing) {
                  s += e;
                  return;
                }
                s += z > za ? e : 0.0;
                w3[2] += z < zb ? e : 0.0;
                if (z <= za && z >= zb && e > 0.0) {
                  w3[1] += e;
                  push(z, i);
                }
              },
              [&](int it) {
                if ((it + 1) % seg_its == 0 || it + 1 == its) {
                  sub[(warp * kSegs + it / seg_its) * 32 + lane] = s;
                  w3[0] += s;
                  s = 0.0;
                }
              });
  };
  bool summed = false;
  int members = 0;  // of rank 0's list that stay, in `sub` not counted
  if (top_p < 1.0) {
    float za, zb;
    propose(true, top_p, true, false, za, zb);
    f64_walk(za, zb, 0.0, true);
    sums(w3);
    const int n = *of_rank(&sh.count, 0);
    sync();
    if (tid == 0) sh.count = 0;
    const double want = top_p * (w3[0] + w3[1] + w3[2]);
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
  if (!summed) {
    __syncthreads();
    f64_walk(-INFINITY, -INFINITY, min_p, false);
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
    int pick = -1, back = -1, n = 0;
    double e[VEC], mine = 0.0;
    walk_part(One(), w, i0, i1,
              [&](float z, uint32_t i) {
                const double x = exp_of(z);
                e[n] = stays(z, i) && x >= min_p ? x : 0.0;
                mine += e[n];
                n++;
              },
              [&](int it) {
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
                    back = (int)first + (w * per_warp + it * 32 + lane) * VEC - shift + j;
                    if (pick < 0 && here > target) pick = back;
                  }
                }
                at += __shfl_sync(0xffffffffu, inc, 31);
                mine = 0.0;
                n = 0;
              });
    const unsigned lowest = __reduce_min_sync(0xffffffffu, (unsigned)pick);
    back = __reduce_max_sync(0xffffffffu, back);
    const int token = lowest != 0xffffffffu ? (int)lowest : back;
    if (lane == 0) {
      float z;
      if constexpr (VEC == 4) z = src[token - first];
      else z = __bfloat162float(src[token - first]);
      a.token[row] = token;
      a.logp[row] = (float)(((double)z - (double)top) / temp - log(total));
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
  // Rows that leave more than half of the places for CTAs (two per SM) empty are split, as long as a part keeps 2,048 values; a part
  // has to fit into shared memory.
  int ranks = 1;
  while (ranks < 8 && a.V > 2048 * ranks && rows * ranks * 2 <= 2 * 148) ranks *= 2;
  while (ranks > 1 && ranks < 8 && (long)a.V * sizeof(T) > 98304L * ranks) ranks *= 2;
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
  PL_REQUIRE(temperature || (temperature_all >= 0.0 && temperature_all <= 1e30), PL_ERR_INVALID, "%s: temperature = %g", me,
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
