// Losses over log-probabilities, with their gradients, and the log-probability of a denoise transition.
//
// All of them are bound by memory: a token costs 2..4 loads, one store and some tens of instructions.  Each reads its
// inputs once and leaves the gradient in the same pass; scalars are summed in float64 per workgroup, in a fixed order,
// and a one-workgroup kernel adds the workgroups' partial sums (no atomics: results do not change from run to run).
#include "finetune.h"
#include "tokens.h"

namespace trebi {

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

// ---------------------------------------------------------------------------------------------------------------
// Valid tokens, where the host does not know them: a mask, lengths, or the mean over sequences (which also needs the
// number of sequences that are not empty).  G lanes take a row, so that rows of 20 tokens and rows of 100 000 both
// keep whole cache lines in flight.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int bytes_set(unsigned x) {       // how many of 4 bytes are not zero
  return __popc((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u);
}
__global__ __launch_bounds__(256) void token_count_kernel(TokenP t, int G, NormPart* np, int* counts) {
  __shared__ double lds[8];
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
        for (long long i = s + gl * 16; i < e; i += G * 16) {
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

// ---------------------------------------------------------------------------------------------------------------
// Clipped policy loss with a KL term
//   d = logp - old, rho = e^d;  beyond a border in the direction that the advantage A pushes, the ratio is held there
//   and the token gives no gradient:   A > 0: d > log(1 + eps_high);  A < 0: d < log(1 - eps_low), or d > log(dual)
//   pg = -A rho;  delta = ref - logp;  kl = -delta | delta^2 / 2 | e^delta - delta - 1
//   loss = sum_i w_i (pg_i + beta kl_i)
// The difference of the log-probabilities and its comparison with the borders are taken in float64, where they are
// exact for every input type: a token does not change sides by a rounding.
// ---------------------------------------------------------------------------------------------------------------
struct PolicyAcc { float pg, kl, rho; int cut, cnt; };

// e^x - 1 and e^x - x - 1 without cancellation: the series below |x| = 1 (its 12th term is under 2^-24 of the sum)
__device__ __forceinline__ void exp_parts(float x, float* em1, float* rest) {
  float q = 1.f / 479001600.f;
  q = fmaf(q, x, 1.f / 39916800.f);
  q = fmaf(q, x, 1.f / 3628800.f);
  q = fmaf(q, x, 1.f / 362880.f);
  q = fmaf(q, x, 1.f / 40320.f);
  q = fmaf(q, x, 1.f / 5040.f);
  q = fmaf(q, x, 1.f / 720.f);
  q = fmaf(q, x, 1.f / 120.f);
  q = fmaf(q, x, 1.f / 24.f);
  q = fmaf(q, x, 1.f / 6.f);
  q = fmaf(q, x, 0.5f);
  float r = x * x * q, m = r + x;
  if (!(fabsf(x) < 1.f)) {
    const float e = expf(x);
    m = e - 1.f;
    r = m - x;
  }
  *em1 = m;
  *rest = r;
}

template <int KL>      // 0: no reference
__device__ __forceinline__ float policy_token(const PolicyP& p, float lp, float old, float ref, float A, float u, float gw,
                                              bool valid, PolicyAcc& a) {
  const double d = (double)lp - (double)old;
  const float rho = expf((float)d);
  const bool over = A > 0.f && d > p.hi, under = A < 0.f && d < p.lo, far = A < 0.f && d > p.dual;
  const bool cut = over || under || far;
  const float held = over ? p.vhi : (under ? p.vlo : p.vdual);
  const float pg = -A * (cut ? held : rho);
  float g = cut ? 0.f : pg, kl = 0.f;
  if (KL) {
    const float x = (float)((double)ref - (double)lp);
    float dk;
    if (KL == 1) { kl = -x; dk = 1.f; }
    else if (KL == 2) { kl = 0.5f * x * x; dk = -x; }
    else { float m; exp_parts(x, &m, &kl); dk = -m; }
    g = fmaf(p.kl_coef, dk, g);
  }
  if (valid) {
    a.pg = fmaf(u, pg, a.pg);
    a.kl = fmaf(u, kl, a.kl);
    a.rho += rho;
    a.cut += cut;
    a.cnt += 1;
  }
  return valid ? g * gw : 0.f;
}

// What multiplies a token besides 1 / (its row's length): 1 / tokens, 1 / sequences or 1 / denominator.
__device__ __forceinline__ double policy_weight(const PolicyP& p, double tokens, double rows) {
  if (p.fixed > 0.0) return p.fixed;
  const double n = p.mode == 0 ? tokens : rows;
  return n > 0.0 ? 1.0 / n : 0.0;
}
template <int NT>
__device__ __forceinline__ double policy_weight_parts(const PolicyP& p, double* lds) {
  if (p.fixed > 0.0) return p.fixed;
  double v[2] = {0, 0};
  for (int i = threadIdx.x; i < p.nnp; i += NT) {
    v[0] += (double)p.np[i].tokens;
    v[1] += (double)p.np[i].rows;
  }
  block_sum<2, NT>(v, lds);
  return policy_weight(p, v[0], v[1]);
}

// The last sequence that begins at or before token i (its first one is 0), searched in [lo, hi].
__device__ __forceinline__ long long find_row(const int* cu, long long lo, long long hi, long long i) {
  while (lo < hi) {
    const long long m = (lo + hi + 1) >> 1;
    if ((long long)cu[m] <= i) lo = m;
    else hi = m - 1;
  }
  return lo;
}

// A row as its tokens see it.
struct RowInfo { long long row, s, e; float A, u, gw; };
template <bool SEQ>
__device__ __forceinline__ void row_info(const PolicyP& p, long long r, double W, const int* counts, RowInfo& ri) {
  ri.row = r;
  row_bounds(p.tk, r, &ri.s, &ri.e);
  ri.A = p.acs ? 0.f : p.adv[r * p.ars];
  if (SEQ) {
    const long long c = counts ? (long long)counts[r] : ri.e - ri.s;
    const double u = c > 0 ? 1.0 / (double)c : 0.0;
    ri.u = (float)u;
    ri.gw = (float)(W * u * (double)p.gscale);
  }
}

// Eight consecutive tokens i .. i + 7 of flat tensors; `ri` is the row of token i.
template <typename T, int KL, bool SEQ, bool PACKED>
__device__ __forceinline__ void policy_eight(const PolicyP& p, long long i, RowInfo ri, double W, const int* counts, double* acc) {
  const long long n = p.tk.n;
  const int m = n - i < 8 ? (int)(n - i) : 8;
  const T *lp = (const T*)p.lp + i, *old = (const T*)(p.old ? p.old : p.lp) + i, *ref = KL ? (const T*)p.ref + i : nullptr;
  float vl[8], vo[8], vr[8], va[8], g[8];
  unsigned valid = 0;
  float A[8], u[8], gw[8];
  long long c = PACKED ? i : i - ri.row * p.tk.len;
  // the tokens' rows
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (PACKED) {
      while (i + e >= ri.e && ri.row + 1 < p.tk.rows) row_info<SEQ>(p, ri.row + 1, W, counts, ri);
      if (i + e >= ri.s && i + e < ri.e) valid |= 1u << e;
    } else {
      if (c >= p.tk.len) {
        c = 0;
        if (e < m) row_info<SEQ>(p, ri.row + 1, W, counts, ri);
      }
      if (c < ri.e) valid |= 1u << e;
      ++c;
    }
    A[e] = ri.A; u[e] = ri.u; gw[e] = ri.gw;
  }
  valid &= (1u << m) - 1u;
  if (p.tk.mask) {
    const unsigned char* mk = p.tk.mask + i;
    if (m == 8) {
      typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(1)));
      const u2 b = *(const TREBI_GLOBAL u2*)mk;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (((e < 4 ? b.x >> (8 * e) : b.y >> (8 * (e - 4))) & 0xffu) == 0) valid &= ~(1u << e);
    } else {
      for (int e = 0; e < m; ++e)
        if (!mk[e]) valid &= ~(1u << e);
    }
  }
  if (valid) {
    if (m == 8) {
      load_vec<8>(lp, vl);
      load_vec<8>(old, vo);
      if (KL) load_vec<8>(ref, vr);
      if (p.acs) load_vec<8>(p.adv + i, va);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = e < m ? e : m - 1;
        vl[e] = load_one(lp + k);
        vo[e] = load_one(old + k);
        if (KL) vr[e] = load_one(ref + k);
        if (p.acs) va[e] = p.adv[i + k];
      }
    }
    PolicyAcc a{0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      g[e] = policy_token<KL>(p, vl[e], vo[e], KL ? vr[e] : 0.f, p.acs ? va[e] : A[e], SEQ ? u[e] : 1.f,
                              SEQ ? gw[e] : (float)(W * (double)p.gscale), (valid >> e) & 1u, a);
    acc[0] += (double)a.pg; acc[1] += (double)a.kl; acc[2] += (double)a.cut; acc[3] += (double)a.rho; acc[4] += (double)a.cnt;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = 0.f;
  }
  if (p.grad) {
    T* o = (T*)p.grad + i;
    if (m == 8) store_vec<8>(o, g);
    else
      for (int e = 0; e < m; ++e) store_one(o + e, g[e]);
  }
}

// One token anywhere (strided views).
template <typename T, int KL, bool SEQ>
__device__ __forceinline__ void policy_one(const PolicyP& p, long long i, double W, const int* counts, double* acc) {
  RowInfo ri;
  long long r, c;
  if (p.tk.n <= 0xffffffffll) {
    r = (unsigned)i / (unsigned)p.tk.len;
    c = (unsigned)i - (unsigned)r * (unsigned)p.tk.len;
  } else {
    r = i / p.tk.len;
    c = i - r * p.tk.len;
  }
  row_info<SEQ>(p, r, W, counts, ri);
  bool valid = c < ri.e;
  if (valid && p.tk.mask) valid = p.tk.mask[r * p.tk.mrs + c * p.tk.mcs] != 0;
  float g = 0.f;
  if (valid) {
    const float lp = load_one((const T*)p.lp + r * p.lrs + c * p.lcs);
    const float old = p.old ? load_one((const T*)p.old + r * p.ors + c * p.ocs) : lp;
    const float ref = KL ? load_one((const T*)p.ref + r * p.rrs + c * p.rcs) : 0.f;
    const float A = p.acs ? p.adv[r * p.ars + c * p.acs] : ri.A;
    PolicyAcc a{0, 0, 0, 0, 0};
    g = policy_token<KL>(p, lp, old, ref, A, SEQ ? ri.u : 1.f, SEQ ? ri.gw : (float)(W * (double)p.gscale), true, a);
    acc[0] += (double)a.pg; acc[1] += (double)a.kl; acc[2] += (double)a.cut; acc[3] += (double)a.rho; acc[4] += (double)a.cnt;
  }
  if (p.grad) store_one((T*)p.grad + i, g);
}

// Tokens [begin, end) by the NT threads of a workgroup.
template <typename T, int KL, bool SEQ, int NT>
__device__ __forceinline__ void policy_range(const PolicyP& p, long long begin, long long end, double W, const int* counts,
                                             double* acc) {
  if (!p.flat) {
    for (long long i = begin + threadIdx.x; i < end; i += NT) policy_one<T, KL, SEQ>(p, i, W, counts, acc);
    return;
  }
  if (p.tk.packed) {
    long long lo = 0;
    for (long long b = begin; b < end; b += NT * 8) {
      const long long last = b + NT * 8 < end ? b + NT * 8 - 1 : end - 1;
      lo = find_row(p.tk.cu, lo, p.tk.rows - 1, b);                     // the same in every thread
      const long long hi = find_row(p.tk.cu, lo, p.tk.rows - 1, last);
      const long long i = b + threadIdx.x * 8;
      if (i < end) {
        RowInfo ri;
        row_info<SEQ>(p, find_row(p.tk.cu, lo, hi, i), W, counts, ri);
        policy_eight<T, KL, SEQ, true>(p, i, ri, W, counts, acc);
      }
    }
  } else {
    for (long long i = begin + threadIdx.x * 8; i < end; i += NT * 8) {
      RowInfo ri;
      const long long r = p.tk.n <= 0xffffffffll ? (long long)((unsigned)i / (unsigned)p.tk.len) : i / p.tk.len;
      row_info<SEQ>(p, r, W, counts, ri);
      policy_eight<T, KL, SEQ, false>(p, i, ri, W, counts, acc);
    }
  }
}

template <typename T, int KL, bool SEQ>
__global__ __launch_bounds__(256) void policy_kernel(PolicyP p) {
  __shared__ double lds[4 * LOSS_VALS];
  const double W = policy_weight_parts<256>(p, lds);
  const long long begin = (long long)blockIdx.x * p.per, end = begin + p.per < p.tk.n ? begin + p.per : p.tk.n;
  double acc[LOSS_VALS] = {0, 0, 0, 0, 0};
  policy_range<T, KL, SEQ, 256>(p, begin, end, W, p.counts, acc);
  block_sum<LOSS_VALS, 256>(acc, lds);
  if (threadIdx.x == 0)
#pragma unroll
    for (int k = 0; k < LOSS_VALS; ++k) p.part[(long long)blockIdx.x * LOSS_VALS + k] = acc[k];
}

__device__ __forceinline__ void policy_stats(const PolicyP& p, const double* v, double W) {
  const double pg = W * v[0], kl = W * v[1], n = v[4] > 0.0 ? v[4] : 1.0;
  p.stats[0] = (float)(pg + (double)p.kl_coef * kl);
  p.stats[1] = (float)pg;
  p.stats[2] = (float)kl;
  p.stats[3] = (float)(v[2] / n);
  p.stats[4] = (float)(v[3] / n);
}

__global__ __launch_bounds__(256) void policy_finish_kernel(PolicyP p, int blocks) {
  __shared__ double lds[4 * LOSS_VALS];
  const double W = policy_weight_parts<256>(p, lds);
  double v[LOSS_VALS] = {0, 0, 0, 0, 0};
  for (int b = threadIdx.x; b < blocks; b += 256)
#pragma unroll
    for (int k = 0; k < LOSS_VALS; ++k) v[k] += p.part[(long long)b * LOSS_VALS + k];
  block_sum<LOSS_VALS, 256>(v, lds);
  if (threadIdx.x == 0) policy_stats(p, v, W);
}

static int group_of(const TokenP& t) {       // lanes a row is given: 16 bytes of mask each
  const long long len = t.packed ? (t.n + t.rows - 1) / t.rows : t.len;
  return !t.mask ? 1 : len <= 64 ? 4 : len <= 512 ? 16 : len <= 4096 ? 64 : 256;
}
hipError_t launch_token_counts(const PolicyP& p, hipStream_t st) {
  hipLaunchKernelGGL(token_count_kernel, dim3(p.nnp), dim3(256), 0, st, p.tk, group_of(p.tk), p.np, p.counts);
  return hipGetLastError();
}
template <typename T>
static hipError_t launch_policy_t(const PolicyP& p, int blocks, hipStream_t st) {
  const int kl = p.ref ? p.kl : 0;
  const bool seq = p.mode == 1;
#define GO(K, S) hipLaunchKernelGGL((policy_kernel<T, K, S>), dim3(blocks), dim3(256), 0, st, p)
  if (seq) { if (kl == 0) GO(0, true); else if (kl == 1) GO(1, true); else if (kl == 2) GO(2, true); else GO(3, true); }
  else { if (kl == 0) GO(0, false); else if (kl == 1) GO(1, false); else if (kl == 2) GO(2, false); else GO(3, false); }
#undef GO
  return hipGetLastError();
}
hipError_t launch_policy(const PolicyP& p, int dtype, int blocks, hipStream_t st) {
  return dtype == 0 ? launch_policy_t<float>(p, blocks, st) : dtype == 1 ? launch_policy_t<bf16_t>(p, blocks, st)
                                                                         : launch_policy_t<f16_t>(p, blocks, st);
}
hipError_t launch_policy_finish(const PolicyP& p, int blocks, hipStream_t st) {
  hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(256), 0, st, p, blocks);
  return hipGetLastError();
}

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
    const float q = expf(-fabsf((float)z)), l1 = log1pf(q), inv = 1.f / (1.f + q);
    const float big = inv, small = q * inv;                              // sigmoid(|z|), sigmoid(-|z|)
    const double pos = (double)l1 + (z < 0 ? -z : 0.0), neg = (double)l1 + (z > 0 ? z : 0.0);   // softplus(-z), softplus(z)
    o.loss = (1.0 - (double)p.smooth) * pos + (p.smooth > 0.f ? (double)p.smooth * neg : 0.0);
    const float sn = z >= 0 ? small : big, sp = z >= 0 ? big : small;    // sigmoid(-z), sigmoid(z)
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

// Sum and number of a row's valid tokens in [s, e), by `G` threads; this thread's part.
template <typename T>
__device__ __forceinline__ void pair_row_sum(const PairP& p, long long r, long long s, long long e, int lane, int G, double* sum,
                                             long long* num) {
  const TokenP& t = p.tk;
  const long long mb = t.packed ? 0 : r * t.mrs, lb = t.packed ? 0 : r * p.lrs, rb = t.packed ? 0 : r * p.rrs;
  const T *lp = (const T*)p.lp + lb, *ref = p.ref ? (const T*)p.ref + rb : nullptr;
  const bool vec = p.lcs == 1 && (!ref || p.rcs == 1);
  double a = 0;
  long long c = 0;
  if (vec) {
    for (long long i = s + lane * 8; i < e; i += (long long)G * 8) {
      const int m = e - i < 8 ? (int)(e - i) : 8;
      const unsigned v = mask_bits(t, mb + i * t.mcs, t.mcs, m);
      if (!v) continue;
      c += __popc(v);
      float x[8], y[8];
      if (m == 8) {
        load_vec<8>(lp + i, x);
        if (ref) load_vec<8>(ref + i, y);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int q = k < m ? k : m - 1;
          x[k] = load_one(lp + i + q);
          if (ref) y[k] = load_one(ref + i + q);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const double d = ref ? (double)x[k] - (double)y[k] : (double)x[k];
        a += (v >> k) & 1u ? d : 0.0;
      }
    }
  } else {
    for (long long i = s + lane; i < e; i += G) {
      if (t.mask && !t.mask[mb + i * t.mcs]) continue;
      const float x = load_one(lp + i * p.lcs);
      a += ref ? (double)x - (double)load_one(ref + i * p.rcs) : (double)x;
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

// G threads take a pair: both rows' sums, the pair, both rows' gradients.  Where there are pairs enough to fill the
// card this is one pass: the gradient needs no second read of the log-probabilities.
template <typename T>
__global__ __launch_bounds__(256) void pairs_whole_kernel(PairP p) {
  __shared__ double lds[16];
  const int G = p.group, per = 256 / G, lane = threadIdx.x & (G - 1), gi = threadIdx.x / G;
  double acc[4] = {0, 0, 0, 0};
  for (long long k0 = (long long)blockIdx.x * per; k0 < p.pairs; k0 += (long long)gridDim.x * per) {
    const long long k = k0 + gi;
    const bool on = k < p.pairs;
    long long s0 = 0, e0 = 0, s1 = 0, e1 = 0, n0 = 0, n1 = 0;
    double v[4] = {0, 0, 0, 0};
    if (on) {
      row_bounds(p.tk, k, &s0, &e0);
      row_bounds(p.tk, k + p.pairs, &s1, &e1);
      pair_row_sum<T>(p, k, s0, e0, lane, G, &v[0], &n0);
      pair_row_sum<T>(p, k + p.pairs, s1, e1, lane, G, &v[2], &n1);
      v[1] = (double)n0;
      v[3] = (double)n1;
    }
    if (G <= 64) {
      for (int o = G >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += __shfl_xor(v[q], o, 64);
    } else {
      block_sum<4, 256>(v, lds);
    }
    if (on) {
      float rc, rr;
      const PairOut o = pair_math(p, k, v[0], v[1], v[2], v[3], &rc, &rr);
      if (lane == 0) {
        p.rew_c[k] = rc;
        p.rew_r[k] = rr;
        acc[0] += o.loss; acc[1] += o.hit; acc[2] += o.z; acc[3] += o.on;
      }
      if (p.grad) {
        pair_row_grad<T>(p, k, s0, e0, p.tk.packed ? e0 : p.tk.len, o.gc, lane, G);
        pair_row_grad<T>(p, k + p.pairs, s1, e1, p.tk.packed ? e1 : p.tk.len, o.gr, lane, G);
      }
    }
  }
  pair_gaps<T>(p);
  block_sum<4, 256>(acc, lds);
  if (threadIdx.x == 0)
    for (int q = 0; q < 4; ++q) p.part[(long long)blockIdx.x * 4 + q] = acc[q];
}

// Few pairs of long rows: `splits` workgroups sum a row, then as many write its gradient.
__device__ __forceinline__ void split_of(long long s, long long e, int splits, int j, long long* a, long long* b) {
  const long long w = ((e - s + splits - 1) / splits + 2047) / 2048 * 2048;      // whole turns of 256 threads x 8 tokens
  *a = s + w * j < e ? s + w * j : e;
  *b = *a + w < e ? *a + w : e;
}
template <typename T>
__global__ __launch_bounds__(256) void pairs_sum_kernel(PairP p) {
  __shared__ double lds[8];
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
  __shared__ double lds[16];
  const long long r = blockIdx.x / p.splits;
  const int j = blockIdx.x - (int)r * p.splits;
  const long long k = r < p.pairs ? r : r - p.pairs;
  double v[4] = {0, 0, 0, 0};
  for (int i = threadIdx.x; i < p.splits; i += 256) {
    const double *c = p.rowpart + (k * p.splits + i) * 2, *q = p.rowpart + ((k + p.pairs) * p.splits + i) * 2;
    v[0] += c[0]; v[1] += c[1]; v[2] += q[0]; v[3] += q[1];
  }
  block_sum<4, 256>(v, lds);
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
__global__ __launch_bounds__(256) void pairs_finish_kernel(PairP p) {
  __shared__ double lds[16];
  double v[4] = {0, 0, 0, 0};
  for (int b = threadIdx.x; b < p.nparts; b += 256)
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += p.part[(long long)b * 4 + q];
  block_sum<4, 256>(v, lds);
  if (threadIdx.x == 0) {
    const double m = v[3] > 0 ? v[3] : 1.0;
    p.stats[0] = (float)(v[0] * p.inv_p);
    p.stats[1] = (float)(v[1] / m);
    p.stats[2] = (float)(v[2] / m);
  }
}

hipError_t launch_pairs_whole(const PairP& p, int dtype, int blocks, hipStream_t st) {
  const dim3 g(blocks), b(256);
  if (dtype == 0) hipLaunchKernelGGL(pairs_whole_kernel<float>, g, b, 0, st, p);
  else if (dtype == 1) hipLaunchKernelGGL(pairs_whole_kernel<bf16_t>, g, b, 0, st, p);
  else hipLaunchKernelGGL(pairs_whole_kernel<f16_t>, g, b, 0, st, p);
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
  hipLaunchKernelGGL(pairs_finish_kernel, dim3(1), dim3(256), 0, st, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// Log-probability of a denoise transition x_t -> x_prev (diffusion.py:153-185, functions.py:131-137: the reverse step
// draws x_prev = mu + sigma z)
//   x0 = pred, or a_t x_t - b_t pred where the net predicts the noise, clamped to [-1, 1] with clip_denoised
//   mu = c1_t x0 + c2_t x_t,  sigma^2 = e^plv_t
//   logp = sum over free elements of -(x_prev - mu)^2 / (2 sigma^2) - (log 2 pi + plv) / 2
//   d logp / d pred = (x_prev - mu) / sigma^2 * c1 * dx0/dpred
// Elements that a condition overwrites are not free, and at t = 0 the step adds no noise: both give 0.
// The residual is a small difference of order-one numbers (sigma falls to 1e-3 of them with long schedules), so it is
// taken in float64; the sum too.
// ---------------------------------------------------------------------------------------------------------------
template <bool BWD, int G>
__global__ __launch_bounds__(256) void transition_kernel(TransP p) {
  __shared__ double lds[4];
  const int lane = threadIdx.x & (G - 1), per = 256 / G;
  const int n = p.H * p.D;
  for (long long b0 = (long long)blockIdx.x * per; b0 < p.B; b0 += (long long)gridDim.x * per) {
    const long long b = b0 + threadIdx.x / G;
    double acc = 0;
    long long tt = 0;
    double plv = 0;
    if (b < p.B) {
      tt = p.t[b];
      tt = tt < 0 ? 0 : (tt >= p.T ? p.T - 1 : tt);
      plv = (double)p.plv[tt];
      const double c1 = (double)p.c1[tt], c2 = (double)p.c2[tt];
      const double ra = p.ra ? (double)p.ra[tt] : 0.0, rm = p.ra ? (double)p.rm[tt] : 0.0;
      double slope = 0;
      if (BWD) slope = (double)p.g[b] * exp(-plv) * c1 * (p.ra ? -rm : 1.0);
      const float *pr = p.pred + b * p.prs, *xt = p.x + b * p.xrs, *xp = p.xp + b * p.xprs;
      float* o = BWD ? p.dpred + b * (long long)n : nullptr;
      for (int i = lane * 4; i < n; i += G * 4) {
        const int m = n - i < 4 ? n - i : 4;
        float vp[4] = {0, 0, 0, 0}, vx[4] = {0, 0, 0, 0}, vq[4] = {0, 0, 0, 0}, d[4] = {0, 0, 0, 0};
        if (tt > 0) {
          if (m == 4) {
            load_vec<4>(pr + i, vp);
            load_vec<4>(xt + i, vx);
            load_vec<4>(xp + i, vq);
          } else {
            for (int e = 0; e < m; ++e) {
              vp[e] = load_one(pr + i + e);
              vx[e] = load_one(xt + i + e);
              vq[e] = load_one(xp + i + e);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            bool free = e < m;
            for (int k = 0; k < p.n_skip; ++k) free = free && !(i + e >= p.skip_lo[k] && i + e < p.skip_hi[k]);
            double x0 = (double)vp[e];
            if (p.ra) x0 = ra * (double)vx[e] - rm * x0;
            bool in = true;
            if (p.clamp) {
              in = !(x0 < -1.0) && !(x0 > 1.0);
              x0 = x0 < -1.0 ? -1.0 : (x0 > 1.0 ? 1.0 : x0);
            }
            const double r = fma(-c1, x0, fma(-c2, (double)vx[e], (double)vq[e]));
            if (BWD) d[e] = free && in ? (float)(r * slope) : 0.f;
            else acc = free ? fma(r, r, acc) : acc;
          }
        }
        if (BWD) {
          if (m == 4) store_vec<4>(o + i, d);
          else
            for (int e = 0; e < m; ++e) store_one(o + i + e, d[e]);
        }
      }
    }
    if (!BWD) {
      if (G == 64) {
        acc = wave_sum64(acc);
      } else {
        double v[1] = {acc};
        block_sum<1, 256>(v, lds);
        acc = v[0];
      }
      if (lane == 0 && b < p.B)
        p.logp[b] = tt > 0 ? (float)(-0.5 * acc * exp(-plv) - p.half_const * (1.8378770664093454836 + plv)) : 0.f;
    }
  }
}
hipError_t launch_transition(const TransP& p, int backward, hipStream_t st) {
  const bool wide = (long long)p.H * p.D > 4096;
  const long long per = wide ? 1 : 4, need = (p.B + per - 1) / per;
  const dim3 g((unsigned)(need < 8192 ? need : 8192)), b(256);
  if (backward) {
    if (wide) hipLaunchKernelGGL((transition_kernel<true, 256>), g, b, 0, st, p);
    else hipLaunchKernelGGL((transition_kernel<true, 64>), g, b, 0, st, p);
  } else {
    if (wide) hipLaunchKernelGGL((transition_kernel<false, 256>), g, b, 0, st, p);
    else hipLaunchKernelGGL((transition_kernel<false, 64>), g, b, 0, st, p);
  }
  return hipGetLastError();
}

}  // namespace trebi
