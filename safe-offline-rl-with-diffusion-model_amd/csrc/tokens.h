// Device helpers of the fine-tuning operators: loads and stores of float32 / bfloat16 / float16 elements at any element
// alignment (gfx950 takes vector accesses at element alignment), and block sums in a fixed order.
#pragma once
#include "device_util.h"

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

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum of K values over a workgroup of NT threads, in every thread; lds: [NT / 64][K].  The order is fixed.
template <int K, int NT>
__device__ __forceinline__ void block_sum(double* v, double* lds) {
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum64(v[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) lds[(threadIdx.x >> 6) * K + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    double a = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) a += lds[w * K + k];
    v[k] = a;
  }
}

}  // namespace trebi
