// Global gradient norm over many tensors, and clipping.
//
//   n = s * (sum_k sum_i g_ki^2)^(1/2)   (or s * sum |g|, or s * max |g|),   c = s * min(1, max_norm / (n + 1e-6)),
//   out = c * g                           s: the factor that takes a loss scale off (1 / loss scale)
//
// Bound by memory: every gradient is read once for the norm and once more (partly still in the 256 MB cache) for the
// scaled copy.  Norm of 1.07 GB of float32: 160 us, 6.7 TB/s.  200 M bfloat16 scaled into float32: 69 us for the norm (400 MB, 5.8
// TB/s) and 247 us for the copy (1.2 GB, 4.9 TB/s, a large copy's rate).  3.96 M float32 into a flat copy: 5.7 and 7.2 us, of which the
// memory takes 6.6: what is left are the launches and the partial sums.  The tensors are cut into chunks on the host and the
// workgroups walk chunks, so that 400 tensors cost the same two launches as one.  The sum is held in float64: no length and no magnitude (1e-30 .. 1e30) loses digits or overflows.
// Each workgroup leaves one partial sum; the kernel that scales adds the partials up itself, every workgroup in the same
// order, so no atomics, no order that changes from run to run, and no third launch.
#include "finetune.h"
#include "tokens.h"

#include <type_traits>

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

// V elements joined to the running values.  Pairs are formed in float32 (one rounding each, 2^-24 of the pair) and added in
// float64: half the float64 work of adding every element, which bfloat16 gradients would otherwise wait for.  Squares
// that leave the middle of float32's range are formed in float64 instead.
template <int NORM, int V>
__device__ __forceinline__ void join_vec(const float* v, double* a0, double* a1) {
  if (NORM == 2) {
    float m = fabsf(v[0]);
    bool nan = v[0] != v[0];
#pragma unroll
    for (int e = 1; e < V; ++e) {
      m = fmaxf(m, fabsf(v[e]));
      nan = nan || v[e] != v[e];
    }
    *a0 = norm_join<2>(*a0, nan ? __builtin_nan("") : (double)m);
    return;
  }
  float q[V / 2], s = 0.f;
#pragma unroll
  for (int e = 0; e < V / 2; ++e) {
    q[e] = NORM == 0 ? fmaf(v[2 * e], v[2 * e], v[2 * e + 1] * v[2 * e + 1]) : fabsf(v[2 * e]) + fabsf(v[2 * e + 1]);
    s += q[e];
  }
  if (s < 1e37f && (NORM == 1 || s > 1e-28f)) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) (e & 1 ? *a1 : *a0) += (double)q[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) *a0 = norm_acc<NORM>(*a0, v[e]);
  }
}

constexpr int DEEP = 8;                               // loads of at most 16 bytes that a thread has in flight

// The `n` elements of a chunk by the workgroup's 256 threads: f(index, values) for whole vectors of V, one(index, value) for
// the few elements behind the last one
template <int V, bool STREAM, typename T, typename F, typename G>
__device__ __forceinline__ void for_vectors(const T* p, int n, F f, G one) {
  constexpr int TURN = DEEP * 256 * V;
  typedef typename Vec<T, V>::type vec;
  const int whole = n & ~(V - 1);
  int base = 0;
  for (; base + TURN <= whole; base += TURN) {
    const int i0 = base + (int)threadIdx.x * V;
    vec r[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const TREBI_GLOBAL vec* q = (const TREBI_GLOBAL vec*)(p + i0 + u * 256 * V);
      r[u] = STREAM ? __builtin_nontemporal_load(q) : *q;
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = up(r[u][e]);
      f(i0 + u * 256 * V, v);
    }
  }
  if (base < whole) {
    const int i0 = base + (int)threadIdx.x * V;
    vec r[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
      if (i0 + u * 256 * V < whole) r[u] = *(const TREBI_GLOBAL vec*)(p + i0 + u * 256 * V);
#pragma unroll
    for (int u = 0; u < DEEP; ++u)
      if (i0 + u * 256 * V < whole) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = up(r[u][e]);
        f(i0 + u * 256 * V, v);
      }
  }
  if (whole + (int)threadIdx.x < n) one(whole + (int)threadIdx.x, load_one(p + whole + threadIdx.x));
}

template <int NORM, bool STREAM>
__global__ __launch_bounds__(256) void grad_partial_kernel(GradP p) {
  __shared__ double lds[4];
  double a0 = 0, a1 = 0;
  auto one = [&](int, float v) { a0 = norm_acc<NORM>(a0, v); };
  for (int c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
    const GradChunk t = uniform_load(p.chunks + c);
    if (t.dtype == 0) for_vectors<4, STREAM>((const float*)t.p, t.len, [&](int, const float* v) { join_vec<NORM, 4>(v, &a0, &a1); }, one);
    else if (t.dtype == 1) for_vectors<8, STREAM>((const bf16_t*)t.p, t.len, [&](int, const float* v) { join_vec<NORM, 8>(v, &a0, &a1); }, one);
    else for_vectors<8, STREAM>((const f16_t*)t.p, t.len, [&](int, const float* v) { join_vec<NORM, 8>(v, &a0, &a1); }, one);
  }
  const double a = block_join<NORM, 256>(norm_join<NORM>(a0, a1), lds);
  if (threadIdx.x == 0) p.part[blockIdx.x] = a;
}

// The norm from the partials, the same in every workgroup that asks.
template <int NT>
__device__ __forceinline__ float grad_total(const GradP& p, double* lds, float* coef) {
  double a = 0;
  if (p.norm_type == 2) {
    for (int i = threadIdx.x; i < p.n_blocks; i += NT) a = norm_join<2>(a, p.part[i]);
    a = block_join<2, NT>(a, lds);
  } else {
    for (int i = threadIdx.x; i < p.n_blocks; i += NT) a += p.part[i];
    a = block_join<0, NT>(a, lds);
    if (p.norm_type == 0) a = sqrt(a);
  }
  const double n = a * (double)p.grad_scale;
  const double c = (double)p.max_norm / (n + 1e-6);
  *coef = (float)((double)p.grad_scale * (c < 1.0 || c != c ? c : 1.0));     // a NaN norm makes every gradient NaN
  return (float)n;
}

__global__ __launch_bounds__(1024) void grad_finish_kernel(GradP p, float* coef_out) {
  __shared__ double lds[16];
  float coef;
  const float n = grad_total<1024>(p, lds, &coef);
  if (threadIdx.x == 0) {
    if (p.norm_out) *p.norm_out = n;
    if (coef_out) *coef_out = coef;
  }
}

template <int V, bool STREAM, typename O>
__device__ __forceinline__ void put_vec(O* p, const float* v) {
  typedef typename Vec<O, V>::type vec;
  vec r;
#pragma unroll
  for (int e = 0; e < V; ++e) r[e] = down<O>(v[e]);
  if (STREAM) __builtin_nontemporal_store(r, (TREBI_GLOBAL vec*)p);
  else *(TREBI_GLOBAL vec*)p = r;
}
template <bool STREAM, typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* p, O* out, int n, float c) {
  constexpr int V = 16 / (int)sizeof(O);               // whole 16-byte stores, neighbouring lanes' next to each other
  for_vectors<V, false>(p, n, [&](int i, float* v) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= c;
    put_vec<V, STREAM>(out + i, v);
  }, [&](int i, float v) { store_one(out + i, v * c); });
}

// The chunks are walked backwards: what the norm's kernel read last is what the cache still holds.
template <bool STREAM>
__global__ __launch_bounds__(256) void grad_scale_kernel(GradP p) {
  __shared__ double lds[4];
  GradChunk t = uniform_load(p.chunks + (p.n_chunks > 0 ? p.n_chunks - 1 - (int)blockIdx.x : 0));
  float c;
  const float norm = grad_total<256>(p, lds, &c);
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.norm_out) *p.norm_out = norm;
  if (!p.out && c == 1.f) return;                     // in place and within the norm: nothing would change
  for (int q = blockIdx.x; q < p.n_chunks; q += gridDim.x) {
    if (q > (int)blockIdx.x) t = uniform_load(p.chunks + p.n_chunks - 1 - q);
    float* o = p.out ? p.out + t.out_off : nullptr;
    if (t.dtype == 0) scale_chunk<STREAM>((const float*)t.p, o ? o : (float*)t.p, t.len, c);
    else if (t.dtype == 1) {
      if (o) scale_chunk<STREAM>((const bf16_t*)t.p, o, t.len, c);
      else scale_chunk<STREAM>((const bf16_t*)t.p, (bf16_t*)t.p, t.len, c);
    } else {
      if (o) scale_chunk<STREAM>((const f16_t*)t.p, o, t.len, c);
      else scale_chunk<STREAM>((const f16_t*)t.p, (f16_t*)t.p, t.len, c);
    }
  }
}

// The same for sets of one chunk a workgroup (up to 8 M elements), which latency bounds: the chunk's loads are on their way
// while the partial sums are added up.  3.96 M float32 into a flat copy 7.2 us, with the kernel above 8.6.
__global__ __launch_bounds__(256) void grad_scale_small_kernel(GradP p) {
  __shared__ double lds[4];
  typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
  const GradChunk t = uniform_load(p.chunks + blockIdx.x);
  const int V = t.dtype == 0 ? 4 : 8, whole = t.len & ~(V - 1), size = t.dtype == 0 ? 4 : 2;
  u4 r[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (u * 256 + (int)threadIdx.x) * V;
    if (i < whole) r[u] = *(const TREBI_GLOBAL u4*)((const char*)t.p + (size_t)i * size);
  }
  float c;
  const float norm = grad_total<256>(p, lds, &c);
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.norm_out) *p.norm_out = norm;
  if (!p.out && c == 1.f) return;
  float* o = p.out ? p.out + t.out_off : nullptr;
  auto put = [&](auto* src, auto* dst) {
    typedef typename std::remove_pointer<decltype(src)>::type T;
    constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = (u * 256 + (int)threadIdx.x) * W;
      if (i < whole) {
        union { u4 q; typename Raw<T>::type e[W]; } x;
        x.q = r[u];
        float v[W];
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = up(x.e[k]) * c;
        store_vec<W>(dst + i, v);
      }
    }
    const int i = whole + (int)threadIdx.x;
    if (i < t.len) store_one(dst + i, load_one(src + i) * c);
  };
  if (t.dtype == 0) put((float*)t.p, o ? o : (float*)t.p);
  else if (t.dtype == 1) {
    if (o) put((bf16_t*)t.p, o);
    else put((bf16_t*)t.p, (bf16_t*)t.p);
  } else {
    if (o) put((f16_t*)t.p, o);
    else put((f16_t*)t.p, (f16_t*)t.p);
  }
}

hipError_t launch_grad_partials(const GradP& p, hipStream_t st) {
  const dim3 g(p.n_blocks), b(256);
#define GO(N)                                                                                  \
  do {                                                                                         \
    if (p.stream_loads) hipLaunchKernelGGL((grad_partial_kernel<N, true>), g, b, 0, st, p);    \
    else hipLaunchKernelGGL((grad_partial_kernel<N, false>), g, b, 0, st, p);                  \
  } while (0)
  if (p.norm_type == 0) GO(0);
  else if (p.norm_type == 1) GO(1);
  else GO(2);
#undef GO
  return hipGetLastError();
}
hipError_t launch_grad_finish(const GradP& p, float* coef_out, hipStream_t st) {
  hipLaunchKernelGGL(grad_finish_kernel, dim3(1), dim3(1024), 0, st, p, coef_out);
  return hipGetLastError();
}
hipError_t launch_grad_scale(const GradP& p, hipStream_t st) {
  if (p.one_each) hipLaunchKernelGGL(grad_scale_small_kernel, dim3(p.n_blocks), dim3(256), 0, st, p);
  else if (p.stream_stores) hipLaunchKernelGGL(grad_scale_kernel<true>, dim3(p.n_blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(grad_scale_kernel<false>, dim3(p.n_blocks), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace trebi
