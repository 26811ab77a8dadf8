// Preference loss over paired log ratios, and its gradient.
//
// Bound by memory where rows are long: 250 pairs of 65536 float32 tokens, 393 MB, 89 us, 4.4 TB/s.  Few or short pairs are
// bound by the launches and one pass of latency (16 pairs of 20 tokens 4.7 us, 512 packed pairs of 1023 10.4), many short ones by the
// pairs' scalars (30000 pairs of 20: 18 us, of which the sigmoid in float64 costs 1.4).  The gradient of a token is the same in its whole row, so it is written, not
// computed; the row has to be summed before.  Sums are taken in float64, in a fixed order, and a one-workgroup kernel adds the
// workgroups' partial sums (2.5 us; no atomics: results do not change from run to run).
#include "finetune.h"
#include "tokens.h"

namespace trebi {

// ---------------------------------------------------------------------------------------------------------------
// Preference loss over pairs of rows: D_r = sum over the row's valid tokens of logp - ref (/ their number),
//   h = D_chosen - D_rejected, z = beta h - margin
//   sigmoid: (1 - e) softplus(-z) + e softplus(z);   hinge: max(0, 1 - z);   ipo: (z / beta - 1 / (2 beta))^2
//   loss = inv_p sum_pairs weight * l;   d loss / d token = +- inv_p weight dl/dh (/ the row's number)
// A pair with an empty row gives nothing.
// ---------------------------------------------------------------------------------------------------------------
struct PairOut { double loss, hit, z, on; float gc, gr; };

__device__ __forceinline__ PairOut pair_math(const PairP& p, long long k, double dc, double nc, double dr, double nr, float* rc,
                                             float* rr) {
  const double sc = p.average ? (nc > 0 ? 1.0 / nc : 0.0) : 1.0, sr = p.average ? (nr > 0 ? 1.0 / nr : 0.0) : 1.0;
  dc *= sc;
  dr *= sr;
  *rc = (float)(p.beta * dc);
  *rr = (float)(p.beta * dr);
  PairOut o{0, 0, 0, 0, 0.f, 0.f};
  if (nc <= 0 || nr <= 0) return o;
  const double h = dc - dr, z = p.beta * h - p.margin;
  double slope;
  if (p.kind == 0) {
    // (in float64: a float32 argument of the exponential, off by |z| 2^-24, would make loss and slope of decided pairs as far off)
    const double q = exp(-fabs(z)), l1 = log1p(q), big = 1.0 / (1.0 + q), small = q * big;      // sigmoid(|z|), sigmoid(-|z|)
    const double pos = l1 + (z < 0 ? -z : 0.0), neg = l1 + (z > 0 ? z : 0.0);                   // softplus(-z), softplus(z)
    o.loss = (1.0 - (double)p.smooth) * pos + (p.smooth > 0.f ? (double)p.smooth * neg : 0.0);
    const double sn = z >= 0 ? small : big, sp = z >= 0 ? big : small;                          // sigmoid(-z), sigmoid(z)
    slope = p.beta * ((double)p.smooth * sp - (1.0 - (double)p.smooth) * sn);
    if (z != z) { o.loss = z; slope = z; }
  } else if (p.kind == 1) {
    o.loss = z >= 1.0 ? 0.0 : 1.0 - z;
    slope = z >= 1.0 ? 0.0 : (z != z ? z : -p.beta);
  } else {
    const double a = (z - 0.5) / p.beta;
    o.loss = a * a;
    slope = 2.0 * a;
  }
  const double w = p.weights ? (double)p.weights[k] : 1.0;
  o.loss *= w;
  o.hit = h > 0 ? 1.0 : 0.0;
  o.z = z;
  o.on = 1.0;
  const double s = slope * w * p.inv_p * (double)p.gscale;
  o.gc = (float)(s * sc);
  o.gr = (float)(-s * sr);
  return o;
}

__device__ __forceinline__ void pair_stats(const PairP& p, const double* v) {
  const double m = v[3] > 0 ? v[3] : 1.0;
  p.stats[0] = (float)(v[0] * p.inv_p);
  p.stats[1] = (float)(v[1] / m);
  p.stats[2] = (float)(v[2] / m);
}

// Eight tokens' validity under the mask (bit e: token i + e), of the first m
__device__ __forceinline__ unsigned mask_bits(const TokenP& t, long long off, long long step, int m) {
  unsigned v = (1u << m) - 1u;
  if (!t.mask) return v;
  if (step == 1 && m == 8) {
    typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(1)));
    const u2 b = *(const TREBI_GLOBAL u2*)(t.mask + off);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (((e < 4 ? b.x >> (8 * e) : b.y >> (8 * (e - 4))) & 0xffu) == 0) v &= ~(1u << e);
  } else {
    for (int e = 0; e < m; ++e)
      if (!t.mask[off + e * step]) v &= ~(1u << e);
  }
  return v;
}

// Sum and number of a row's valid tokens in [s, e), by `G` threads; this thread's part.  16 tokens a thread on their way.
// Differences are taken in float64, where they are exact.
template <typename T>
__device__ __forceinline__ void pair_row_sum(const PairP& p, long long r, long long s, long long e, int lane, int G, double* sum,
                                             long long* num) {
  const TokenP& t = p.tk;
  const long long mb = t.packed ? 0 : r * t.mrs, lb = t.packed ? 0 : r * p.lrs, rb = t.packed ? 0 : r * p.rrs;
  const T *lp = (const T*)p.lp + lb, *ref = p.ref ? (const T*)p.ref + rb : nullptr;
  double a = 0;
  long long c = 0;
  if (p.lcs == 1 && (!ref || p.rcs == 1)) {
    const long long step = (long long)G * 8;
    for (long long i0 = s + lane * 8; i0 < e; i0 += 2 * step) {
      unsigned v[2];
      Pack<T, 8> x[2], y[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long i = i0 + h * step;
        v[h] = i + 8 <= e ? mask_bits(t, mb + i * t.mcs, t.mcs, 8) : 0u;
        if (v[h]) {
          x[h].load(lp + i);
          if (ref) y[h].load(ref + i);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        c += __popc(v[h]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool on = (v[h] >> k) & 1u;
          a += (double)(on ? x[h].at(k) : 0.f) - (double)(on && ref ? y[h].at(k) : 0.f);
        }
      }
    }
    // the last tokens, fewer than 8: one a lane
    const long long i = s + (e > s ? (e - s) / 8 * 8 : 0) + lane;
    if (lane < 8 && i < e && (!t.mask || t.mask[mb + i * t.mcs])) {
      a += (double)load_one(lp + i) - (ref ? (double)load_one(ref + i) : 0.0);
      ++c;
    }
  } else {
    for (long long i = s + lane; i < e; i += G) {
      if (t.mask && !t.mask[mb + i * t.mcs]) continue;
      const float x = load_one(lp + i * p.lcs);
      a += (double)x - (ref ? (double)load_one(ref + i * p.rcs) : 0.0);
      ++c;
    }
  }
  *sum = a;
  *num = c;
}

// The gradient of a row's positions [s, e), of which [s, ve) may be valid
template <typename T>
__device__ __forceinline__ void pair_row_grad(const PairP& p, long long r, long long s, long long ve, long long e, float g, int lane,
                                              int G) {
  const TokenP& t = p.tk;
  const long long mb = t.packed ? 0 : r * t.mrs;
  T* o = (T*)p.grad + (t.packed ? 0 : r * t.len);
  for (long long i = s + lane * 8; i < e; i += (long long)G * 8) {
    const int m = e - i < 8 ? (int)(e - i) : 8;
    const int mv = ve <= i ? 0 : ve - i < m ? (int)(ve - i) : m;
    const unsigned v = mv ? mask_bits(t, mb + i * t.mcs, t.mcs, mv) : 0u;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (v >> k) & 1u ? g : 0.f;
    if (m == 8) store_vec<8>(o + i, x);
    else
      for (int k = 0; k < m; ++k) store_one(o + i + k, x[k]);
  }
}

// Packed tokens of no sequence: before the first and behind the last
template <typename T>
__device__ __forceinline__ void pair_gaps(const PairP& p) {
  if (!p.tk.packed || !p.grad) return;
  long long a = p.tk.cu[0], b = p.tk.cu[p.tk.rows];
  a = a < 0 ? 0 : (a > p.tk.n ? p.tk.n : a);
  b = b < a ? a : (b > p.tk.n ? p.tk.n : b);
  const long long me = (long long)blockIdx.x * blockDim.x + threadIdx.x, all = (long long)gridDim.x * blockDim.x;
  for (long long i = me; i < a; i += all) store_one((T*)p.grad + i, 0.f);
  for (long long i = b + me; i < p.tk.n; i += all) store_one((T*)p.grad + i, 0.f);
}

// G threads take a pair, half of them a row: the rows' sums, the pair, the rows' gradients.  Where there are pairs enough
// to fill the card this is one pass: the gradient needs no second read of the log-probabilities.  A workgroup takes 256 / G
// pairs and ends: in a loop over pairs the compiler kept what does not change in registers, 190 of them (8000 pairs of 200
// float32 tokens, 64 threads each: 27 us, now 19).  Four waves a SIMD: with five the 16-bit kernels spill and gain nothing.
template <typename T, int G>
__global__ __launch_bounds__(256, 4) void pairs_whole_kernel(PairP p) {
  __shared__ double lds[20];
  constexpr int half = G >> 1, per = 256 / G;
  const int gi = threadIdx.x / G, lane = threadIdx.x & (half - 1);
  const bool second = threadIdx.x & half;
  const long long k = (long long)blockIdx.x * per + gi, r = second ? k + p.pairs : k;
  const bool on = k < p.pairs;
  double acc[4] = {0, 0, 0, 0}, v[2] = {0, 0}, o[2];
  long long s = 0, e = 0, n = 0;
  if (on) {
    row_bounds(p.tk, r, &s, &e);
    pair_row_sum<T>(p, r, s, e, lane, half, &v[0], &n);
    v[1] = (double)n;
  }
  if (G <= 64) {
#pragma unroll
    for (int q = half >> 1; q > 0; q >>= 1) {
      v[0] += __shfl_xor(v[0], q, 64);
      v[1] += __shfl_xor(v[1], q, 64);
    }
    o[0] = __shfl_xor(v[0], half, 64);
    o[1] = __shfl_xor(v[1], half, 64);
  } else {                                            // the workgroup takes one pair, half of its waves a row
    constexpr int HW = 2;
    v[0] = wave_sum64(v[0]);
    v[1] = wave_sum64(v[1]);
    if ((threadIdx.x & 63) == 0) {
      lds[(threadIdx.x >> 6) * 2] = v[0];
      lds[(threadIdx.x >> 6) * 2 + 1] = v[1];
    }
    __syncthreads();
    const int mine = second ? 2 * HW : 0, other = 2 * HW - mine;
    v[0] = v[1] = o[0] = o[1] = 0.0;
#pragma unroll
    for (int w = 0; w < HW; ++w) {
      v[0] += lds[mine + 2 * w];
      v[1] += lds[mine + 2 * w + 1];
      o[0] += lds[other + 2 * w];
      o[1] += lds[other + 2 * w + 1];
    }
  }
  if (on) {
    float rc, rr;
    const PairOut q = pair_math(p, k, second ? o[0] : v[0], second ? o[1] : v[1], second ? v[0] : o[0], second ? v[1] : o[1], &rc, &rr);
    if (lane == 0 && !second) {
      p.rew_c[k] = rc;
      p.rew_r[k] = rr;
      acc[0] = q.loss; acc[1] = q.hit; acc[2] = q.z; acc[3] = q.on;
    }
    if (p.grad) pair_row_grad<T>(p, r, s, e, p.tk.packed ? e : p.tk.len, second ? q.gr : q.gc, lane, half);
  }
  pair_gaps<T>(p);
  if (per > 1) block_sum<4, 256>(acc, lds);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) pair_stats(p, acc);
    else
      for (int q = 0; q < 4; ++q) p.part[(long long)blockIdx.x * 4 + q] = acc[q];
  }
}

// Few pairs of long rows: `splits` workgroups sum a row, then as many write its gradient.  24 pairs of 131072 float32 tokens, 63 MB:
// 9.8 us for the sums, 9.3 for the gradient (25 MB: bound by the latency of the parts it begins with).
__device__ __forceinline__ void split_of(long long s, long long e, int splits, int j, long long* a, long long* b) {
  const long long w = ((e - s + splits - 1) / splits + 511) / 512 * 512;         // whole waves of 8 tokens a lane
  *a = s + w * j < e ? s + w * j : e;
  *b = *a + w < e ? *a + w : e;
}
template <typename T>
__global__ __launch_bounds__(256) void pairs_sum_kernel(PairP p) {
  __shared__ double lds[10];
  const long long r = blockIdx.x / p.splits;
  const int j = blockIdx.x - (int)r * p.splits;
  long long s, e, a, b, n;
  row_bounds(p.tk, r, &s, &e);
  split_of(s, e, p.splits, j, &a, &b);
  double v[2];
  pair_row_sum<T>(p, r, a, b, threadIdx.x, 256, &v[0], &n);
  v[1] = (double)n;
  block_sum<2, 256>(v, lds);
  if (threadIdx.x == 0) {
    p.rowpart[(long long)blockIdx.x * 2] = v[0];
    p.rowpart[(long long)blockIdx.x * 2 + 1] = v[1];
  }
}
template <typename T>
__global__ __launch_bounds__(256) void pairs_grad_kernel(PairP p) {
  const long long r = blockIdx.x / p.splits;
  const int j = blockIdx.x - (int)r * p.splits;
  const long long k = r < p.pairs ? r : r - p.pairs;
  double v[4] = {0, 0, 0, 0};                          // every wave adds the splits' sums up for itself: no barrier
  for (int i = threadIdx.x & 63; i < p.splits; i += 64) {
    const double *c = p.rowpart + (k * p.splits + i) * 2, *q = p.rowpart + ((k + p.pairs) * p.splits + i) * 2;
    v[0] += c[0]; v[1] += c[1]; v[2] += q[0]; v[3] += q[1];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = wave_sum64(v[q]);
  float rc, rr;
  const PairOut o = pair_math(p, k, v[0], v[1], v[2], v[3], &rc, &rr);
  if (r < p.pairs && j == 0 && threadIdx.x == 0) {
    p.rew_c[k] = rc;
    p.rew_r[k] = rr;
    double* d = p.part + k * 4;
    d[0] = o.loss; d[1] = o.hit; d[2] = o.z; d[3] = o.on;
  }
  if (!p.grad) return;
  long long s, ve, a, b;
  row_bounds(p.tk, r, &s, &ve);
  split_of(s, p.tk.packed ? ve : p.tk.len, p.splits, j, &a, &b);
  pair_row_grad<T>(p, r, a, ve, b, r < p.pairs ? o.gc : o.gr, threadIdx.x, 256);
  pair_gaps<T>(p);
}
__global__ __launch_bounds__(1024) void pairs_finish_kernel(PairP p) {
  __shared__ double lds[17 * 4];
  double v[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int b = threadIdx.x; b < p.nparts; b += 1024)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += p.part[(long long)b * 4 + q];
  block_sum<4, 1024>(v, lds);
  if (threadIdx.x == 0) pair_stats(p, v);
}

hipError_t launch_pairs_whole(const PairP& p, int dtype, hipStream_t st) {
  const dim3 g(p.nparts), b(256);
#define GO(T)                                                                                          \
  do {                                                                                                 \
    if (p.group == 16) hipLaunchKernelGGL((pairs_whole_kernel<T, 16>), g, b, 0, st, p);                \
    else if (p.group == 64) hipLaunchKernelGGL((pairs_whole_kernel<T, 64>), g, b, 0, st, p);           \
    else hipLaunchKernelGGL((pairs_whole_kernel<T, 256>), g, b, 0, st, p);                             \
  } while (0)
  if (dtype == 0) GO(float);
  else if (dtype == 1) GO(bf16_t);
  else GO(f16_t);
#undef GO
  return hipGetLastError();
}
template <typename T>
static hipError_t launch_pairs_split_t(const PairP& p, hipStream_t st) {
  const dim3 g((unsigned)(p.tk.rows * p.splits)), b(256);
  hipLaunchKernelGGL(pairs_sum_kernel<T>, g, b, 0, st, p);
  if (hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(pairs_grad_kernel<T>, g, b, 0, st, p);
  return hipGetLastError();
}
hipError_t launch_pairs_split(const PairP& p, int dtype, hipStream_t st) {
  return dtype == 0 ? launch_pairs_split_t<float>(p, st) : dtype == 1 ? launch_pairs_split_t<bf16_t>(p, st)
                                                                      : launch_pairs_split_t<f16_t>(p, st);
}
hipError_t launch_pairs_finish(const PairP& p, hipStream_t st) {
  hipLaunchKernelGGL(pairs_finish_kernel, dim3(1), dim3(1024), 0, st, p);
  return hipGetLastError();
}

}  // namespace trebi
