// Clipped policy loss with a KL term: token counts, the sum of the workgroups' parts, and which kernel a call takes (the kernels
// themselves: policy.inl).
#include "finetune.h"
#include "tokens.h"

namespace trebi {

// ---------------------------------------------------------------------------------------------------------------
// Valid tokens, where the host does not know them: a mask, lengths, or the mean over sequences (which also needs the
// number of sequences that are not empty).  Bound by latency: 4096 lengths 4 us, a mask of 512 x 2047 2.7 us.  G lanes take a row, so that rows of 20 tokens and rows of 100 000 both
// keep whole cache lines in flight.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int bytes_set(unsigned x) {       // how many of 4 bytes are not zero
  return __popc((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u);
}
__global__ __launch_bounds__(256) void token_count_kernel(TokenP t, int G, NormPart* np, int* counts) {
  __shared__ double lds[10];
  const int per = 256 / G, gl = threadIdx.x & (G - 1), gi = threadIdx.x / G;
  long long tokens = 0, used = 0;
  for (long long r0 = (long long)blockIdx.x * per; r0 < t.rows; r0 += (long long)gridDim.x * per) {
    const long long r = r0 + gi;
    long long c = 0;
    if (r < t.rows) {
      long long s, e;
      row_bounds(t, r, &s, &e);
      if (!t.mask) c = gl == 0 ? e - s : 0;
      else if (t.mcs == 1) {
        const unsigned char* m = t.mask + (t.packed ? 0 : r * t.mrs);
        typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(1)));
        const long long step = (long long)G * 16;
        long long i = s + gl * 16;
        for (; i + 3 * step + 16 <= e; i += 4 * step) {           // (few long rows: four loads on their way)
          u4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = *(const TREBI_GLOBAL u4*)(m + i + u * step);
#pragma unroll
          for (int u = 0; u < 4; ++u) c += bytes_set(v[u].x) + bytes_set(v[u].y) + bytes_set(v[u].z) + bytes_set(v[u].w);
        }
        for (; i < e; i += step) {
          if (i + 16 <= e) {
            const u4 v = *(const TREBI_GLOBAL u4*)(m + i);
            c += bytes_set(v.x) + bytes_set(v.y) + bytes_set(v.z) + bytes_set(v.w);
          } else {
            for (long long j = i; j < e; ++j) c += m[j] != 0;
          }
        }
      } else {
        for (long long i = s + gl; i < e; i += G) c += t.mask[r * t.mrs + i * t.mcs] != 0;
      }
    }
    if (G <= 64) {
      for (int o = G >> 1; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    } else {                                        // G == 256: one row a workgroup
      double v[1] = {(double)c};                    // exact below 2^53
      block_sum<1, 256>(v, lds);
      c = (long long)v[0];
    }
    if (gl == 0 && r < t.rows) {
      if (counts) counts[r] = (int)(c > 0x7fffffff ? 0x7fffffff : c);
      tokens += c;
      used += c > 0;
    }
  }
  double v[2] = {(double)tokens, (double)used};
  block_sum<2, 256>(v, lds);
  if (threadIdx.x == 0) np[blockIdx.x] = {(long long)v[0], (long long)v[1]};
}

// Lanes a row is given: 16 bytes of mask each
static int group_of(const TokenP& t) {
  const long long len = t.packed ? (t.n + t.rows - 1) / t.rows : t.len;
  return !t.mask ? 1 : len <= 64 ? 4 : len <= 256 ? 16 : len <= 1024 ? 64 : 256;
}
// Where only the tokens of a contiguous mask are wanted, between the first and the last offset, rows do not matter
__global__ __launch_bounds__(256) void mask_count_kernel(TokenP t, NormPart* np) {
  __shared__ double lds[5];
  typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(1)));
  long long s = 0, e = t.n;
  if (t.packed) {
    s = uniform_load(t.cu);
    e = uniform_load(t.cu + t.rows);
    s = s < 0 ? 0 : s;
    e = e > t.n ? t.n : e;
  }
  const unsigned char* m = t.mask;
  const long long step = (long long)gridDim.x * 4096;
  long long c = 0;
  for (long long i = s + ((long long)blockIdx.x * 256 + threadIdx.x) * 16; i < e; i += step) {
    if (i + 16 <= e) {
      const u4 v = *(const TREBI_GLOBAL u4*)(m + i);
      c += bytes_set(v.x) + bytes_set(v.y) + bytes_set(v.z) + bytes_set(v.w);
    } else {
      for (long long j = i; j < e; ++j) c += m[j] != 0;
    }
  }
  double v[1] = {(double)c};
  block_sum<1, 256>(v, lds);
  if (threadIdx.x == 0) np[blockIdx.x] = {(long long)v[0], 0};
}
hipError_t launch_token_counts(PolicyP& p, hipStream_t st) {
  const TokenP& t = p.tk;
  const bool whole = t.mask && !t.lengths && p.mode == 0 && (t.packed || (t.mcs == 1 && t.mrs == t.len));
  const long long want = whole ? (t.n + 4095) / 4096 : t.mask ? t.rows : (t.rows + 255) / 256;
  p.nnp = (int)(want < COUNT_BLOCKS ? want : COUNT_BLOCKS);
  if (whole) hipLaunchKernelGGL(mask_count_kernel, dim3(p.nnp), dim3(256), 0, st, t, p.np);
  else
    hipLaunchKernelGGL(token_count_kernel, dim3(p.nnp), dim3(256), 0, st, t, group_of(t), p.np, p.counts);
  return hipGetLastError();
}
hipError_t launch_policy_f32(const PolicyP& p, int blocks, hipStream_t st);
hipError_t launch_policy_bf16(const PolicyP& p, int blocks, hipStream_t st);
hipError_t launch_policy_f16(const PolicyP& p, int blocks, hipStream_t st);
hipError_t launch_policy(const PolicyP& p, int dtype, int blocks, hipStream_t st) {
  return dtype == 0 ? launch_policy_f32(p, blocks, st) : dtype == 1 ? launch_policy_bf16(p, blocks, st) : launch_policy_f16(p, blocks, st);
}

__global__ __launch_bounds__(1024) void policy_finish_kernel(PolicyP p, int blocks) {
  __shared__ double lds[17 * LOSS_VALS];
  double v[LOSS_VALS] = {0, 0, 0, 0, 0};
  for (int b = threadIdx.x; b < blocks; b += 1024)
#pragma unroll
    for (int k = 0; k < LOSS_VALS; ++k) v[k] += p.part[k * LOSS_PARTS + b];
  block_sum<LOSS_VALS, 1024>(v, lds);
  if (threadIdx.x == 0) policy_stats(p, v, blocks ? *p.weight : 0.0);
}

hipError_t launch_policy_finish(const PolicyP& p, int blocks, hipStream_t st) {
  hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(1024), 0, st, p, blocks);
  return hipGetLastError();
}

}  // namespace trebi
