// Device helpers of the fine-tuning operators: loads and stores of float32 / bfloat16 / float16 elements at any element
// alignment (gfx950 takes vector accesses at element alignment), and block sums in a fixed order.
#pragma once
#include "device_util.h"
#include "finetune.h"

namespace trebi {

struct bf16_t { unsigned short u; };
typedef _Float16 f16_t;

template <typename T> struct Raw;
template <> struct Raw<float> { typedef float type; };
template <> struct Raw<bf16_t> { typedef unsigned short type; };
template <> struct Raw<f16_t> { typedef _Float16 type; };
template <typename T, int V> struct Vec {
  typedef typename Raw<T>::type raw;
  typedef raw type __attribute__((ext_vector_type(V), aligned(sizeof(raw))));
};

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(_Float16 v) { return (float)v; }
__device__ __forceinline__ float up(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
// rounded once, to nearest even
template <typename T> __device__ __forceinline__ typename Raw<T>::type down(float v);
template <> __device__ __forceinline__ float down<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 down<f16_t>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ unsigned short down<bf16_t>(float v) {
  union { __bf16 b; unsigned short u; } c;
  c.b = (__bf16)v;
  return c.u;
}

template <typename T>
__device__ __forceinline__ float load_one(const T* p) {
  return up(*(const TREBI_GLOBAL typename Raw<T>::type*)p);
}
template <typename T>
__device__ __forceinline__ void store_one(T* p, float v) {
  *(TREBI_GLOBAL typename Raw<T>::type*)p = down<T>(v);
}
// V consecutive elements, as at most 16-byte accesses
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  constexpr int W = V * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
  typedef typename Vec<T, W>::type vec;
#pragma unroll
  for (int k = 0; k < V; k += W) {
    const vec r = *(const TREBI_GLOBAL vec*)(p + k);
#pragma unroll
    for (int e = 0; e < W; ++e) v[k + e] = up(r[e]);
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  constexpr int W = V * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
  typedef typename Vec<T, W>::type vec;
#pragma unroll
  for (int k = 0; k < V; k += W) {
    vec r;
#pragma unroll
    for (int e = 0; e < W; ++e) r[e] = down<T>(v[k + e]);
    *(TREBI_GLOBAL vec*)(p + k) = r;
  }
}

// N consecutive elements as they lie in memory: loaded first, widened when they are needed, so that the loads of a turn are
// all on their way before the first of them is waited for.
template <typename T, int N> struct Pack {
  static constexpr int W = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
  typename Vec<T, W>::type r[N / W];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < N / W; ++k) r[k] = *(const TREBI_GLOBAL typename Vec<T, W>::type*)(p + k * W);
  }
  __device__ __forceinline__ float at(int e) const { return up(r[e / W][e % W]); }
};

// Loads through the scalar cache, at an index that is the same in every lane of the wave and from memory that nothing
// writes while the kernel runs.  They are counted apart from the vector loads, which return in order: a look-up by vector
// loads would wait for all the data asked for before it.
template <typename T>
__device__ __forceinline__ T uniform_load(const T* p) {
  if constexpr (sizeof(T) <= 8) {
    return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
  } else {                                             // a struct of 8-byte words
    union { T t; long long w[sizeof(T) / 8]; } c;
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 8; ++k) c.w[k] = ((const __attribute__((address_space(4))) long long*)(uintptr_t)p)[k];
    return c.t;
  }
}
__device__ __forceinline__ long long uniform(long long v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v);
  const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)((unsigned long long)v >> 32));
  return (long long)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  union { double d; int i[2]; } c, r;
  c.d = v;
  r.i[0] = __builtin_amdgcn_update_dpp(0, c.i[0], CTRL, 0xf, 0xf, false);
  r.i[1] = __builtin_amdgcn_update_dpp(0, c.i[1], CTRL, 0xf, 0xf, false);
  return r.d;
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  union { double d; int i[2]; } c, r;
  c.d = v;
  r.i[0] = __builtin_amdgcn_readlane(c.i[0], lane);
  r.i[1] = __builtin_amdgcn_readlane(c.i[1], lane);
  return r.d;
}
// Sum over the wave's 64 lanes (all of them active), in every lane; exchanges inside the registers, in a fixed order
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp_d<0xB1>(v);      // quad_perm [1,0,3,2]
  v += dpp_d<0x4E>(v);      // quad_perm [2,3,0,1]
  v += dpp_d<0x141>(v);     // row_half_mirror
  v += dpp_d<0x140>(v);     // row_mirror
  return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
// Sum of K values over a workgroup of NT threads, in a fixed order; lds: [NT / 64 + 1][K].  In every thread up to 256
// threads, in thread 0 of a larger workgroup.
template <int K, int NT>
__device__ __forceinline__ void block_sum(double* v, double* lds) {
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum64(v[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) lds[(threadIdx.x >> 6) * K + k] = v[k];
  __syncthreads();
  if (NT <= 256) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      double a = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) a += lds[w * K + k];
      v[k] = a;
    }
  } else {
    if (threadIdx.x < K) {
      double a = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) a += lds[w * K + threadIdx.x];
      lds[(NT / 64) * K + threadIdx.x] = a;            // the first wave's own: no barrier
    }
    if (threadIdx.x == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = lds[(NT / 64) * K + k];
  }
}

// Tokens [*s, *e) of row r, as columns (padded) or flat positions (packed); offsets that leave the buffer are cut.
__device__ __forceinline__ void row_bounds(const TokenP& t, long long r, long long* s, long long* e) {
  if (t.packed) {
    long long a = t.cu[r], b = t.cu[r + 1];
    a = a < 0 ? 0 : (a > t.n ? t.n : a);
    *s = a;
    *e = b < a ? a : (b > t.n ? t.n : b);
  } else {
    *s = 0;
    long long b = t.lengths ? (long long)t.lengths[r] : t.len;
    *e = b < 0 ? 0 : (b > t.len ? t.len : b);
  }
}

// The policy loss's scalars from its sums (pg, kl, cut, rho, count) and the weight
__device__ __forceinline__ void policy_stats(const PolicyP& p, const double* v, double W) {
  const double pg = W * v[0], kl = W * v[1], n = v[4] > 0.0 ? v[4] : 1.0;
  p.stats[0] = (float)(pg + (double)p.kl_coef * kl);
  p.stats[1] = (float)pg;
  p.stats[2] = (float)kl;
  p.stats[3] = (float)(v[2] / n);
  p.stats[4] = (float)(v[3] / n);
}

}  // namespace trebi
