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
// A row is read once: a cluster of CTAs holds it in shared memory, each a contiguous slice, and what follows are passes
// over that. The borders of top-k and top-p are found by a descent: 32 bins of d = max - z (equal steps; f32, every step
// of it monotone, so a bin's members all come before the next one's), the bin in which the count or the mass is
// reached, 32 bins of that, until its members fit a list, which is sorted. Each thread has its own 32 bins (no atomics:
// their order would change the f64 sums). Logits with more equals than the list holds end in a search over the keys' bits.
#include <cooperative_groups.h>

#include "pl_common.cuh"
#include "pl_runtime.h"

namespace cg = cooperative_groups;

namespace pl {

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 32, kList = 2048, kLevels = 4;
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

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }

// An unsigned key that orders like the value; both zeros have one key.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// 2^y for y <= 0: 2^(n/16) from a table, 2^r, |r| <= 1/32, by its series (the next term is 5e-16 of the value).
__device__ __forceinline__ double exp2_neg(double y, const double* tab) {
  if (!(y > -1020.0)) return 0.0;
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the rounded integer
  const double s = fma(y, 16.0, magic);
  const int n = __double2loint(s);
  const double r = fma(s - magic, -0.0625, y);
  const double l = 0.6931471805599453094;
  double q = l * l * l * l * l * l / 720.0;
  q = fma(q, r, l * l * l * l * l / 120.0);
  q = fma(q, r, l * l * l * l / 24.0);
  q = fma(q, r, l * l * l / 6.0);
  q = fma(q, r, l * l / 2.0);
  q = fma(q, r, l);
  q = fma(q, r, 1.0) * tab[n & 15];
  return __hiloint2double(__double2hiint(q) + (n >> 4) * (1 << 20), __double2loint(q));
}

__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  double bins[2][kBins];  // what the cluster's CTAs read of one another, by turns
  double warp[kWarps];
  double tab[16];
  float fwarp[kWarps][3];
  float top[2][3];
  double above, total;
  int chosen, count, found;
  uint32_t tkey, tidx;
  int tie[kWarps];
};

// The bin descent's levels: an element is above, in or below the region that they describe.
struct Region {
  int levels;
  float lo[kLevels], inv[kLevels];
  int bin[kLevels];
  __device__ __forceinline__ static int bin_of(float d, float lo, float inv) {
    return (int)fminf(fmaxf((d - lo) * inv, 0.f), (float)(kBins - 1));
  }
  __device__ __forceinline__ int where(float d) const {
#pragma unroll
    for (int l = 0; l < kLevels; l++) {
      if (l >= levels) break;
      const int b = bin_of(d, lo[l], inv[l]);
      if (b != bin[l]) return b < bin[l] ? -1 : 1;
    }
    return 0;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  grid_wait();
  grid_next();
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char mem[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  double* hist = reinterpret_cast<double*>(mem);                      // [kBins][kThreads]
  unsigned long long* list = reinterpret_cast<unsigned long long*>(mem);  // [kList], of rank 0, in its place
  T* z = reinterpret_cast<T*>(mem + sizeof(double) * kBins * kThreads);

  // ---- the row's options
  const double t_given = a.temp ? (double)a.temp[row] : a.temp0, p_given = a.p ? (double)a.p[row] : a.p0;
  const double mp_given = a.min_p ? (double)a.min_p[row] : a.min_p0;
  const double u_given = (double)a.u[row];
  int k = a.k ? a.k[row] : a.k0;
  double temp = t_given, top_p = p_given, min_p = fmin(mp_given, 1.0);
  const double u = fmin(fmax(u_given, 0.0), 1.0);
  const bool fine = t_given >= 0.0 && t_given < INFINITY && p_given == p_given && mp_given == mp_given && u_given == u_given;
  if (temp == 0.0 || top_p <= 0.0) k = 1;  // the first in order alone
  if (k == 1) {
    temp = 1.0;
    top_p = 1.0;
    min_p = 0.0;
  }
  if (k <= 0 || k >= a.V) k = 0;
  const double c = 1.4426950408889634074 / temp;  // e = 2^(c (z - max))

  // ---- the slice into shared memory, its start kept at the same offset from a 16-byte boundary; around it -inf
  const long first = (long)rank * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  const int len = last > first ? (int)(last - first) : 0;
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + first;
  const int shift = len ? (int)(((uintptr_t)src & 15) / sizeof(T)) : 0;
  const int vecs = (shift + len + VEC - 1) / VEC;
  const int per_warp = (vecs + kWarps * 32 - 1) / (kWarps * 32) * 32;  // a warp's vectors lie together
  float top = -INFINITY, nan = 0.f;
  for (int it = 0; it < per_warp; it += 32) {
    const int v = warp * per_warp + it + lane;
    if (v >= vecs) continue;
    __align__(16) T x[VEC];
    const int at = v * VEC - shift;
    if (at >= 0 && at + VEC <= len) {
      *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(src + at));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) x[j] = at + j >= 0 && at + j < len ? src[at + j] : (T)(-INFINITY);
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const float f = value(x[j]);
      top = fmaxf(top, f);
      if (f != f) nan = 1.f;
    }
    *reinterpret_cast<uint4*>(z + v * VEC) = *reinterpret_cast<const uint4*>(x);
  }
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
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; w++) {
      top = fmaxf(top, sh.fwarp[w][0]);
      nan = fmaxf(nan, sh.fwarp[w][1]);
    }
    sh.top[0][0] = top;
    sh.top[0][1] = nan;
    sh.count = 0;
  }
  cluster.sync();
  top = -INFINITY, nan = 0.f;
  for (int q = 0; q < ranks; q++) {
    const float* other = cluster.map_shared_rank(&sh.top[0][0], q);
    top = fmaxf(top, other[0]);
    nan = fmaxf(nan, other[1]);
  }
  if (!fine || nan != 0.f || fabsf(top) == INFINITY) {  // the same for every CTA of the cluster
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      a.logp[row] = __int_as_float(0x7fffffff);
    }
    cluster.sync();
    return;
  }

  const double max_z = (double)top;
  auto exp_of = [&](float f) { return exp2_neg(((double)f - max_z) * c, sh.tab); };
  // f(value, index in the row) for every value of the slice, a warp's in ascending order
  auto each = [&](auto f) {
    for (int it = 0; it < per_warp; it += 32) {
      const int v = warp * per_warp + it + lane;
      if (v >= vecs) continue;
      __align__(16) T x[VEC];
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(z + v * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j++) f(value(x[j]), (uint32_t)(first + v * VEC - shift + j));
    }
  };
  int turn = 0;
  // One number per CTA to the cluster's sum, added in rank order (every thread gets it); `before`: what lower ranks have.
  auto cluster_sum = [&](double v, double* before) {
    v = warp_add(v);
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int w = 0; w < kWarps; w++) s += sh.warp[w];
      sh.bins[turn][0] = s;
    }
    cluster.sync();
    double s = 0.0;
    for (int q = 0; q < ranks; q++) {
      if (q == rank && before) *before = s;
      s += *cluster.map_shared_rank(&sh.bins[turn][0], q);
    }
    turn ^= 1;
    return s;
  };

  // ---- the border (tkey, tidx) of what stays: key > tkey, or key = tkey and index <= tidx
  uint32_t tkey = 0, tidx = 0xffffffffu;
  auto stays = [&](uint32_t key, uint32_t i) { return key > tkey || (key == tkey && i <= tidx); };

  // Sorts the n entries of rank 0's list (called by all of its threads); n rounded up to a power of two with ~0.
  auto sort_list = [&](int n) {
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
    return size;
  };
  auto list_exp = [&](unsigned long long e) {  // of an entry (~key, index)
    const uint32_t key = ~(uint32_t)(e >> 32);
    return exp_of(__uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key));
  };
  // Exclusive sums over the list in its order, thread t's eight entries from 8 t; `total` of all.
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
    if (lane == 31) sh.warp[warp] = inc;
    __syncthreads();
    double base = 0.0;
    total = 0.0;
    for (int w = 0; w < kWarps; w++) {
      if (w == warp) base = total;
      total += sh.warp[w];
    }
    __syncthreads();
    const double up = __shfl_up_sync(0xffffffffu, inc, 1);
    return base + (lane ? up : 0.0);
  };

  // The descent. by_mass: up to the share `want` (in mass if it is given, else in tokens) among those that stay so far.
  // In list_all, the list gets the members and all above them.
  auto descend = [&](bool by_mass, double want, bool share, bool list_all, float range) {
    Region reg;
    reg.levels = 0;
    float lo = 0.f, hi = range;
    double above = 0.0;  // weight of what is surely kept
    bool listed = false;
    const float end = 750.f * (float)fmin(temp, 1e35);  // beyond it every e is zero
    for (int level = 0; level < kLevels && !listed; level++) {
      const float inv = fminf((float)kBins / fmaxf(hi - lo, 1e-37f), 1e30f);
      for (int b = 0; b < kBins; b++) hist[b * kThreads + tid] = 0.0;
      each([&](float f, uint32_t i) {
        const float d = top - f;
        if (!(d <= end) || reg.where(d) != 0) return;
        if (by_mass && !stays(key_of(f), i)) return;
        const int b = Region::bin_of(d, lo, inv);
        hist[b * kThreads + tid] += by_mass ? exp_of(f) : 1.0;
      });
      __syncthreads();
      for (int b = warp; b < kBins; b += kWarps) {
        double s = 0.0;
        for (int q = 0; q < kThreads / 32; q++) s += hist[b * kThreads + q * 32 + lane];
        s = warp_add(s);
        if (lane == 0) sh.bins[turn][b] = s;
      }
      cluster.sync();
      if (tid < 32) {
        double s = 0.0;
        for (int q = 0; q < ranks; q++) s += *cluster.map_shared_rank(&sh.bins[turn][tid], q);
        hist[tid] = s;  // every thread's bins have been added up
      }
      turn ^= 1;
      __syncthreads();
      if (tid == 0) {
        if (share && level == 0) {
          double total = 0.0;
          for (int b = 0; b < kBins; b++) total += hist[b];
          want *= total;
        }
        int b = 0, some = 0;
        double at = above, at_some = above;
        for (; b < kBins; b++) {
          if (hist[b] > 0.0) some = b, at_some = at;
          if (at + hist[b] >= want) break;
          at += hist[b];
        }
        if (b == kBins || hist[b] == 0.0) b = some, at = at_some;  // short of it by rounding, or of members: the last ones
        sh.chosen = b;
        sh.above = at;
        sh.total = want;
        if (rank == 0) sh.count = 0;
      }
      __syncthreads();
      above = sh.above;
      want = sh.total;
      reg.lo[level] = lo;
      reg.inv[level] = inv;
      reg.bin[level] = sh.chosen;
      reg.levels = level + 1;
      const float w = 1.f / inv, from = lo + sh.chosen * w;
      if (sh.chosen == kBins - 1) hi = fmaxf(hi, level ? lo + kBins * w : end);
      else hi = from + w;
      lo = from;
      cluster.sync();  // rank 0's bins are free: its list may be written, from a count of zero
      int* count = cluster.map_shared_rank(&sh.count, 0);
      unsigned long long* to = cluster.map_shared_rank(list, 0);
      each([&](float f, uint32_t i) {
        const float d = top - f;
        const uint32_t key = key_of(f);
        if (!(d <= end)) return;
        const int side = reg.where(d);
        if (side > 0 || (side < 0 && !list_all) || !stays(key, i)) return;
        const int n = atomicAdd(count, 1);
        if (n < kList) to[n] = (unsigned long long)(~key) << 32 | i;
      });
      cluster.sync();
      listed = *cluster.map_shared_rank(&sh.count, 0) <= kList;
    }
    const int n = listed ? *cluster.map_shared_rank(&sh.count, 0) : 0;
    if (listed) {
      if (!list_all) {
        if (rank == 0) {
          sort_list(n);
          double e[8], total;
#pragma unroll
          for (int j = 0; j < 8; j++) e[j] = 8 * tid + j < n ? (by_mass ? list_exp(list[8 * tid + j]) : 1.0) : 0.0;
          double at = above + list_scan(e, total);
          int mine = -1;  // the last that less than `want` comes before
#pragma unroll
          for (int j = 0; j < 8; j++) {
            if (8 * tid + j < n && (at < want || 8 * tid + j == 0)) mine = 8 * tid + j;
            at += e[j];
          }
          mine = __reduce_max_sync(0xffffffffu, mine);
          if (lane == 0) sh.tie[warp] = mine;
          __syncthreads();
          if (tid == 0) {
            for (int w = 0; w < kWarps; w++) mine = max(mine, sh.tie[w]);
            sh.tkey = mine >= 0 ? ~(uint32_t)(list[mine] >> 32) : 0u;
            sh.tidx = mine >= 0 ? (uint32_t)list[mine] : 0xffffffffu;
          }
        }
        cluster.sync();
        const uint32_t key = *cluster.map_shared_rank(&sh.tkey, 0), idx = *cluster.map_shared_rank(&sh.tidx, 0);
        tkey = key;
        tidx = idx;
        cluster.sync();
      }
      return n;
    }
    // More members than the list holds, after the last level: equal or nearly equal logits. The largest key whose
    // members from it on reach `want`, bit by bit; then so many of its equals as are needed, the lowest indices first.
    auto weight_from = [&](uint32_t from) {
      double s = 0.0;
      each([&](float f, uint32_t i) {
        const float d = top - f;
        const uint32_t key = key_of(f);
        if (key < from || !(d <= end) || reg.where(d) != 0 || !stays(key, i)) return;
        s += by_mass ? exp_of(f) : 1.0;
      });
      return cluster_sum(s, nullptr);
    };
    want = fmin(want, above + weight_from(0));
    uint32_t key = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if (above + weight_from(key | bit) >= want) key |= bit;
    if (key != 0xffffffffu) above += weight_from(key + 1);
    double mine = 0.0, before;
    each([&](float f, uint32_t i) {
      if (key_of(f) == key && reg.where(top - f) == 0 && stays(key, i)) mine += 1.0;
    });
    const double own = warp_add(mine), equals = cluster_sum(mine, &before);
    const float f = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    const double each_w = by_mass ? exp_of(f) : 1.0;
    double need = fmin(fmax(ceil((want - above) / each_w), 1.0), equals);
    if (above + (need - 1.0) * each_w >= want && need > 1.0) need -= 1.0;  // the quotient's rounding
    // the need-th equal: the rank, warp, step and lane that hold it
    if (tid == 0) sh.found = -1;
    if (lane == 0) sh.warp[warp] = own;
    __syncthreads();
    for (int w = 0; w < warp; w++) before += sh.warp[w];
    if (before < need && need <= before + own) {
      for (int it = 0; it < per_warp; it += 32) {
        const int v = warp * per_warp + it + lane;
        int n = 0;
        if (v < vecs)
          for (int j = 0; j < VEC; j++) {
            const float g = value(z[v * VEC + j]);
            n += key_of(g) == key && reg.where(top - g) == 0 && stays(key, (uint32_t)(first + v * VEC - shift + j));
          }
        int inc = n;
        for (int o = 1; o < 32; o *= 2) {
          const int up = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += up;
        }
        const double from = before + (double)(inc - n);
        if (from < need && need <= from + (double)n) {
          int left = (int)(need - from);
          for (int j = 0; j < VEC; j++) {
            const float g = value(z[v * VEC + j]);
            const uint32_t i = (uint32_t)(first + v * VEC - shift + j);
            if (key_of(g) == key && reg.where(top - g) == 0 && stays(key, i) && --left == 0) sh.found = (int)i;
          }
        }
        before += (double)__shfl_sync(0xffffffffu, inc, 31);
      }
    }
    cluster.sync();
    int found = -1;
    for (int q = 0; q < ranks; q++) found = max(found, *cluster.map_shared_rank(&sh.found, q));
    cluster.sync();
    tkey = key;
    tidx = (uint32_t)found;
    return -1;
  };

  if (k > 0) {
    // steps of the logits' own spread: twice the mean distance from the largest, far ones (e = 0) counting as 750 T
    const float end = 750.f * (float)fmin(temp, 1e35);
    double s = 0.0;
    each([&](float f, uint32_t i) { s += i < (uint32_t)last && i >= (uint32_t)first ? (double)fminf(top - f, end) : 0.0; });
    const float range = (float)(2.0 * cluster_sum(s, nullptr) / a.V);
    const bool few = k <= kList / 2;
    const int n = descend(false, (double)k, false, few, range);
    if (few && n >= 0) {  // the list holds all of the first k: the rest is rank 0's
      if (rank == 0) {
        sort_list(n);
        const int m = n < k ? n : k;
        double e[8], total;
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = 8 * tid + j < m ? list_exp(list[8 * tid + j]) : 0.0;
        double at = list_scan(e, total);
        // top-p and min-p end the sorted list somewhere: what goes is moved to its end, the rest sorted by index
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
          const uint32_t key = (uint32_t)mine[j];
          e[j] = mine[j] == ~0ull ? 0.0 : list_exp((unsigned long long)(~key) << 32);
        }
        at = list_scan(e, total);
        const double target = u * total;
        int pick = -1, back = -1;  // the first whose sum passes the target; the last with any mass
#pragma unroll
        for (int j = 0; j < 8; j++) {
          at += e[j];
          if (e[j] > 0.0) {
            back = 8 * tid + j;
            if (pick < 0 && at > target) pick = 8 * tid + j;
          }
        }
        const unsigned first_pick = __reduce_min_sync(0xffffffffu, (unsigned)pick);
        back = __reduce_max_sync(0xffffffffu, back);
        if (lane == 0) {
          sh.tie[warp] = (int)first_pick;
          sh.fwarp[warp][0] = __int_as_float(back);
        }
        __syncthreads();
        if (tid == 0) {
          unsigned best = 0xffffffffu;
          for (int w = 0; w < kWarps; w++) {
            best = min(best, (unsigned)sh.tie[w]);
            back = max(back, __float_as_int(sh.fwarp[w][0]));
          }
          const unsigned long long e1 = list[best != 0xffffffffu ? (int)best : back];
          const uint32_t key = (uint32_t)e1;
          const float f = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
          a.token[row] = (int)(e1 >> 32);
          a.logp[row] = (float)(((double)f - max_z) / temp - log(total));
        }
      }
      cluster.sync();
      return;
    }
    // list_all ended in the search over bits, or the border alone is known
  }
  if (top_p < 1.0) descend(true, top_p, true, false, 24.f * (float)fmin(temp, 1e35));

  // ---- the draw: sums by warp, then the warp that holds u's place walks its part once more
  double s = 0.0;
  auto mass = [&](float f, uint32_t i) {
    if (!stays(key_of(f), i)) return 0.0;
    const double e = exp_of(f);
    return e >= min_p ? e : 0.0;
  };
  each([&](float f, uint32_t i) { s += mass(f, i); });
  const double own = warp_add(s);
  const double total = cluster_sum(s, nullptr);
  const double target = u * total;
  // u's place is in the last rank, and there in the last warp, that has any mass and does not begin behind it; where
  // rounding (or u = 1) leaves the target unreached there, its last kept token is the one
  int holder = -1;
  double before = 0.0, from = 0.0;
  for (int q = 0; q < ranks; q++) {
    const double part = *cluster.map_shared_rank(&sh.bins[turn ^ 1][0], q);
    if (part > 0.0 && from <= target) holder = q, before = from;
    from += part;
  }
  if (lane == 0) sh.warp[warp] = own;
  __syncthreads();
  int held = -1;
  from = before;
  for (int w = 0; w < kWarps; w++) {
    const double part = sh.warp[w];
    if (part > 0.0 && from <= target) held = w, before = from;
    from += part;
  }
  int pick = -1, back = -1;
  if (rank == holder && warp == held)
    for (int it = 0; it < per_warp; it += 32) {
      const int v = warp * per_warp + it + lane;
      double e[VEC], n = 0.0;
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        e[j] = v < vecs ? mass(value(z[v * VEC + j]), (uint32_t)(first + v * VEC - shift + j)) : 0.0;
        n += e[j];
      }
      double inc = n;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const double up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const double up = __shfl_up_sync(0xffffffffu, inc, 1);
      double at = before + (lane ? up : 0.0);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        at += e[j];
        if (e[j] > 0.0) {
          back = (int)(first + v * VEC - shift + j);
          if (pick < 0 && at > target) pick = back;
        }
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  if (rank == holder && warp == held) {
    const unsigned lowest = __reduce_min_sync(0xffffffffu, (unsigned)pick);
    back = __reduce_max_sync(0xffffffffu, back);
    const int token = lowest != 0xffffffffu ? (int)lowest : back;
    if (lane == 0) {
      a.token[row] = token;
      a.logp[row] = (float)(((double)value(z[token - first + shift]) - max_z) / temp - log(total));
    }
  }
  cluster.sync();
}

template <typename T>
static int sample_launch(SampleArgs& a, long rows, cudaStream_t st) {
  // A cluster's CTAs share a row. Slices of at most 32 KB leave room for two CTAs on an SM beside their bins; few rows
  // are split further, down to 2,048 values, so that more SMs work on them.
  int ranks = 1;
  while (ranks < 8 && ((long)a.V * sizeof(T) > 32768L * ranks || (rows * ranks * 2 <= 148 && a.V > 2048 * ranks))) ranks *= 2;
  a.slice = (int)round_up(ceil_div(a.V, ranks), 8);
  const size_t smem = sizeof(double) * kBins * kThreads + ((size_t)a.slice * sizeof(T) + 32);
  int rc = raise_smem((const void*)sample_kernel<T>, smem);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(rows * ranks);
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  PL_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<T>, (const SampleArgs)a));
  count_launch();
  return PL_OK;
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
