// What the row kernels (pl_norm.cu, pl_block.cu) share: vectors of values in registers, their two-lane f32 arithmetic and
// the sums over the threads that own a row.
#pragma once
#include "pl_common.cuh"

namespace pl {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// VEC consecutive values of type T as they lie in memory. Rows are read and written once: streaming accesses, so
// that the weights stay in L1.
template <typename T, int VEC>
struct __align__(sizeof(T) * VEC) Pack {
  T v[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * VEC == 16) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
      *reinterpret_cast<uint4*>(v) = u;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) v[j] = __ldcs(p + j);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) * VEC == 16) {
      __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(v));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j++) __stcs(p + j, v[j]);
    }
  }
};
template <int VEC>
__device__ __forceinline__ void load_param(const float* __restrict__ p, long c, float (&o)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + c + j));
      o[j] = f.x;
      o[j + 1] = f.y;
      o[j + 2] = f.z;
      o[j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o[j] = __ldg(p + c + j);
  }
}

// Sums and products over the VEC values of a vector, two lanes at a time where VEC is even (sm_100's two-lane f32
// instructions; both kernels are bound by instruction issue before HBM otherwise).
template <int VEC>
struct Vec {
  float v[VEC];
  __device__ __forceinline__ float2 at(int j) const { return make_float2(v[j], v[j + 1]); }
  __device__ __forceinline__ void set(int j, float2 f) {
    v[j] = f.x;
    v[j + 1] = f.y;
  }
};
template <typename T, int VEC>
__device__ __forceinline__ Vec<VEC> widen(const Pack<T, VEC>& p) {
  Vec<VEC> o;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.v);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      o.v[j] = __uint_as_float(w[j / 2] << 16);
      o.v[j + 1] = __uint_as_float(w[j / 2] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = to_f(p.v[j]);
  }
  return o;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> narrow(const Vec<VEC>& f) {
  Pack<T, VEC> o;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(o.v);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[j], f.v[j + 1]);
      w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = from_f<T>(f.v[j]);
  }
  return o;
}
// a b + c, a + b, a b on every value
template <int VEC>
__device__ __forceinline__ Vec<VEC> vfma(const Vec<VEC>& a, const Vec<VEC>& b, const Vec<VEC>& c) {
  Vec<VEC> o;
  if constexpr (VEC % 2 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) o.set(j, __ffma2_rn(a.at(j), b.at(j), c.at(j)));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = __fmaf_rn(a.v[j], b.v[j], c.v[j]);
  }
  return o;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> vadd(const Vec<VEC>& a, const Vec<VEC>& b) {
  Vec<VEC> o;
  if constexpr (VEC % 2 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) o.set(j, __fadd2_rn(a.at(j), b.at(j)));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = a.v[j] + b.v[j];
  }
  return o;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> vmul(const Vec<VEC>& a, const Vec<VEC>& b) {
  Vec<VEC> o;
  if constexpr (VEC % 2 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) o.set(j, __fmul2_rn(a.at(j), b.at(j)));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) o.v[j] = a.v[j] * b.v[j];
  }
  return o;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> vall(float f) {
  Vec<VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; j++) o.v[j] = f;
  return o;
}
template <int VEC>
__device__ __forceinline__ float vsum(const Vec<VEC>& a) {
  float s = a.v[0];
#pragma unroll
  for (int j = 1; j < VEC; j++) s += a.v[j];
  return s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the TPR threads of a row group (a fixed order). `scr` holds 32 floats of the block's own for this call.
template <int TPR>
__device__ __forceinline__ float group_sum(float v, float* scr) {
  v = warp_sum(v);
  if constexpr (TPR == 32) return v;
  constexpr int NW = TPR / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) scr[warp] = v;
  __syncthreads();
  const int w0 = warp / NW * NW;
  return warp_sum(lane < NW ? scr[w0 + lane] : 0.f);
}

// Threads of a block whose rows take TPR threads each, and the blocks that share an SM.
__host__ __device__ constexpr int norm_threads(int tpr) { return tpr > 256 ? tpr : 256; }
__host__ __device__ constexpr int norm_blocks(int tpr) { return tpr > 256 ? 1 : 2; }

// Sums N values (a power of two up to 32) over the lanes with one exchange less per level than the values kept:
// lane l returns the total of value l / (32 / N).
template <int N>
__device__ __forceinline__ float warp_sum_n(const float (&v)[N], int lane) {
  if constexpr (N == 1) {
    return warp_sum(v[0]);
  } else {
    float a[N / 2];
    constexpr int OFF = 16;
    const bool hi = lane & OFF;
#pragma unroll
    for (int j = 0; j < N / 2; j++) {
      const float send = hi ? v[j] : v[j + N / 2], keep = hi ? v[j + N / 2] : v[j];
      a[j] = keep + __shfl_xor_sync(0xffffffffu, send, OFF);
    }
    if constexpr (N == 2) {
      float c = a[0];
#pragma unroll
      for (int o = 8; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
      return c;
    } else {
      float b[N / 4];
      const bool hi2 = lane & 8;
#pragma unroll
      for (int j = 0; j < N / 4; j++) {
        const float send = hi2 ? a[j] : a[j + N / 4], keep = hi2 ? a[j + N / 4] : a[j];
        b[j] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
      }
      float c = b[0];
      if constexpr (N == 8) {
        const bool hi3 = lane & 4;
        const float send = hi3 ? b[0] : b[1], keep = hi3 ? b[1] : b[0];
        c = keep + __shfl_xor_sync(0xffffffffu, send, 4);
      } else {
        c += __shfl_xor_sync(0xffffffffu, c, 4);
      }
      c += __shfl_xor_sync(0xffffffffu, c, 2);
      c += __shfl_xor_sync(0xffffffffu, c, 1);
      return c;
    }
  }
}

// Totals over each row group of the N values a thread brings (a fixed order), the values spread over the lanes: lane l
// of every warp of the group holds value l / (32 / N). `scr` is [N][32] floats that no thread still reads.
template <int TPR, int N>
__device__ __forceinline__ float group_sum_n(const float (&s)[N], float (*scr)[32], int lane, int warp) {
  constexpr int NW = TPR / 32, LV = 32 / N;
  float v = warp_sum_n<N>(s, lane);
  if constexpr (NW > 1) {
    if (lane % LV == 0) scr[lane / LV][warp] = v;
    __syncthreads();
    v = 0.f;
    const int w0 = warp / NW * NW;
#pragma unroll
    for (int q = 0; q < (NW + LV - 1) / LV; q++)
      if (lane % LV + LV * q < NW) v += scr[lane / LV][w0 + lane % LV + LV * q];
#pragma unroll
    for (int o = 1; o < LV; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

constexpr int kNormSms = 148;             // SMs that the persistent grids are sized for
constexpr int kNormParts = 2 * kNormSms;  // most blocks (and slices) whose column sums are kept

static inline bool vec_ok(const void* p, size_t ld, size_t esz) {
  return ((uintptr_t)p & 15) == 0 && (ld * esz) % 16 == 0;
}

// dw[c] = sum_p part[p][0][c], db[c] = sum_p part[p][1][c] in the order of the parts (pl_norm.cu).
int param_launch(const float* part, int parts, long cols, float* dw, float* db, cudaStream_t st);

}  // namespace pl
