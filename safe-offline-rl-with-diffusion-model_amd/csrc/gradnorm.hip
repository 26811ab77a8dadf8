// Global gradient norm over many tensors, and clipping.
//
//   n = s * (sum_k sum_i g_ki^2)^(1/2)   (or s * sum |g|, or s * max |g|),   c = s * min(1, max_norm / (n + 1e-6)),
//   out = c * g                           s: the factor that takes a loss scale off (1 / loss scale)
//
// Bound by memory: every gradient is read once for the norm and once more (partly still in the 256 MB cache) for the
// scaled copy.  The tensors are cut into chunks on the host; a workgroup walks chunks, so that 400 tensors cost the
// same two launches as one.  The sum is taken in float64: the card converts and adds doubles at half the float rate,
// several times faster than HBM delivers, and then no length and no magnitude (1e-30 .. 1e30) loses digits or
// overflows.  Each workgroup leaves one partial sum; the kernel that scales adds the partials up itself, every
// workgroup in the same order, so no atomics, no order that changes from run to run, and no third launch.
#include "finetune.h"
#include "tokens.h"

namespace trebi {

template <int NORM>
__device__ __forceinline__ double norm_join(double a, double b) {
  if (NORM != 2) return a + b;
  return a != a ? a : (b > a || b != b ? b : a);      // a NaN wins and stays
}
template <int NORM>
__device__ __forceinline__ double norm_acc(double a, float v) {
  if (NORM == 0) return fma((double)v, (double)v, a);
  return norm_join<NORM>(a, (double)fabsf(v));
}

template <int NORM, int NT>
__device__ __forceinline__ double block_join(double a, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = norm_join<NORM>(a, __shfl_xor(a, o, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  a = lds[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) a = norm_join<NORM>(a, lds[w]);
  return a;
}

template <int NORM, typename T>
__device__ __forceinline__ double chunk_norm(const T* p, int len) {
  constexpr int V = 16 / sizeof(T);                   // one 16-byte load
  double a0 = 0, a1 = 0;
  int i = threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= len; i += 4 * 256 * V) {   // four loads in flight
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_vec<V>(p + i + u * 256 * V, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        a0 = norm_acc<NORM>(a0, v[u][e]);
        a1 = norm_acc<NORM>(a1, v[u][e + 1]);
      }
  }
  for (; i < len; i += 256 * V) {
    if (i + V <= len) {
      float v[V];
      load_vec<V>(p + i, v);
#pragma unroll
      for (int e = 0; e < V; ++e) a0 = norm_acc<NORM>(a0, v[e]);
    } else {
      for (int e = i; e < len; ++e) a0 = norm_acc<NORM>(a0, load_one(p + e));
    }
  }
  return norm_join<NORM>(a0, a1);
}

template <int NORM>
__global__ __launch_bounds__(256) void grad_partial_kernel(GradP p) {
  __shared__ double lds[4];
  double a = 0;
  for (int c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
    const GradChunk ch = p.chunks[c];
    const GradTensor t = p.tensors[ch.tensor];
    double v;
    if (t.dtype == 0) v = chunk_norm<NORM>((const float*)t.p + ch.off, ch.len);
    else if (t.dtype == 1) v = chunk_norm<NORM>((const bf16_t*)t.p + ch.off, ch.len);
    else v = chunk_norm<NORM>((const f16_t*)t.p + ch.off, ch.len);
    a = norm_join<NORM>(a, v);
  }
  a = block_join<NORM, 256>(a, lds);
  if (threadIdx.x == 0) p.part[blockIdx.x] = a;
}

// The norm from the partials, the same in every workgroup that asks.
__device__ __forceinline__ float grad_total(const GradP& p, double* lds, float* coef) {
  double a = 0;
  if (p.norm_type == 2) {
    for (int i = threadIdx.x; i < p.n_part; i += 256) a = norm_join<2>(a, p.part[i]);
    a = block_join<2, 256>(a, lds);
  } else {
    for (int i = threadIdx.x; i < p.n_part; i += 256) a += p.part[i];
    a = block_join<0, 256>(a, lds);
    if (p.norm_type == 0) a = sqrt(a);
  }
  const double n = a * (double)p.grad_scale;
  const double c = (double)p.max_norm / (n + 1e-6);
  *coef = (float)((double)p.grad_scale * (c < 1.0 || c != c ? c : 1.0));     // a NaN norm makes every gradient NaN
  return (float)n;
}

__global__ __launch_bounds__(256) void grad_finish_kernel(GradP p, float* coef_out) {
  __shared__ double lds[4];
  float coef;
  const float n = grad_total(p, lds, &coef);
  if (threadIdx.x == 0) {
    if (p.norm_out) *p.norm_out = n;
    if (coef_out) *coef_out = coef;
  }
}

template <typename T, typename O>
__device__ __forceinline__ void chunk_scale(const T* p, O* out, int len, float c) {
  constexpr int V = 16 / sizeof(T);
  int i = threadIdx.x * V;
  for (; i + 3 * 256 * V + V <= len; i += 4 * 256 * V) {
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_vec<V>(p + i + u * 256 * V, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[u][e] *= c;
      store_vec<V>(out + i + u * 256 * V, v[u]);
    }
  }
  for (; i < len; i += 256 * V) {
    if (i + V <= len) {
      float v[V];
      load_vec<V>(p + i, v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= c;
      store_vec<V>(out + i, v);
    } else {
      for (int e = i; e < len; ++e) store_one(out + e, load_one(p + e) * c);
    }
  }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(GradP p) {
  __shared__ double lds[4];
  float c;
  const float n = grad_total(p, lds, &c);
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.norm_out) *p.norm_out = n;
  if (!p.out && c == 1.f) return;                     // in place and within the norm: nothing would change
  for (int k = blockIdx.x; k < p.n_chunks; k += gridDim.x) {
    const GradChunk ch = p.chunks[k];
    const GradTensor t = p.tensors[ch.tensor];
    float* o = p.out ? p.out + t.out_off + ch.off : nullptr;
    if (t.dtype == 0) {
      const float* g = (const float*)t.p + ch.off;
      chunk_scale(g, o ? o : (float*)g, ch.len, c);
    } else if (t.dtype == 1) {
      const bf16_t* g = (const bf16_t*)t.p + ch.off;
      if (o) chunk_scale(g, o, ch.len, c);
      else chunk_scale(g, (bf16_t*)g, ch.len, c);
    } else {
      const f16_t* g = (const f16_t*)t.p + ch.off;
      if (o) chunk_scale(g, o, ch.len, c);
      else chunk_scale(g, (f16_t*)g, ch.len, c);
    }
  }
}

hipError_t launch_grad_partials(const GradP& p, hipStream_t st) {
  const dim3 g(p.n_part), b(256);
  if (p.norm_type == 0) hipLaunchKernelGGL(grad_partial_kernel<0>, g, b, 0, st, p);
  else if (p.norm_type == 1) hipLaunchKernelGGL(grad_partial_kernel<1>, g, b, 0, st, p);
  else hipLaunchKernelGGL(grad_partial_kernel<2>, g, b, 0, st, p);
  return hipGetLastError();
}
hipError_t launch_grad_finish(const GradP& p, float* coef_out, hipStream_t st) {
  hipLaunchKernelGGL(grad_finish_kernel, dim3(1), dim3(256), 0, st, p, coef_out);
  return hipGetLastError();
}
hipError_t launch_grad_scale(const GradP& p, hipStream_t st) {
  hipLaunchKernelGGL(grad_scale_kernel, dim3(p.n_part), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace trebi
