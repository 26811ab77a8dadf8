// Clipped policy loss with a KL term, and its gradient: the kernels, for one element type (policy_f32.hip and its likes).
//
// A token costs 2..4 loads, one store and some tens of instructions.  4.2 M packed float32 tokens, three inputs, an advantage a token,
// a gradient: 83 MB, 25.7 us, 3.2 TB/s; the vector units issue 42 % of the time.  4096 x 8192 padded bfloat16 tokens, of which 0.75 count,
// second KL term: 218 MB, 60 us, 3.7 TB/s; 60 vector instructions for each 64 tokens that count, which the vector units issue in 61 % of
// the time.  Inputs are read once and the gradient leaves in the same pass; scalars are summed in float64, in a fixed order, and a
// one-workgroup kernel adds the workgroups' partial sums (4 us; no atomics: results do not change from run to run).
#include "finetune.h"
#include "tokens.h"

namespace trebi {

// ---------------------------------------------------------------------------------------------------------------
// Clipped policy loss with a KL term
//   d = logp - old, rho = e^d;  beyond a border in the direction that the advantage A pushes, the ratio is held there
//   and the token gives no gradient:   A > 0: d > log(1 + eps_high);  A < 0: d < log(1 - eps_low), or d > log(dual)
//   pg = -A rho;  delta = ref - logp;  kl = -delta | delta^2 / 2 | e^delta - delta - 1
//   loss = sum_i w_i (pg_i + beta kl_i)
// A thread takes N = 16 bytes of consecutive tokens (4 or 8).  N tokens of rows of at least N lie in at most two rows, so
// what belongs to a row (advantage, borders, weight) is looked up twice, not N times, and a wave whose tokens all count and
// lie in one row runs without any selection: with 8 bytes a token (bfloat16) it is the instructions that would bound this
// kernel.  Which row that is goes through the scalar cache, beside the loads of the tokens themselves; for packed sequences
// the wave looks for it 64 offsets at a time (two loads for 4096 sequences, where halving takes twelve).
// A token's side of a border must not hang on a rounding.  d is rounded to float32, which cannot carry it past the
// border's own float32 value but can make the two equal; only then the comparison is made again in float64, where the
// difference is exact for every input type.
// ---------------------------------------------------------------------------------------------------------------
// Sums are float64 from the token on: many tokens are held at the same border, or hold the same ratio, and float32 sums of the same
// few values round the same way again and again (9e-8 of eight equal terms, which advantages of both signs do not hide).
struct PolicySum { double pg, kl, rho; unsigned cut, cnt; };      // (a thread has fewer than 2^31 of 2^46 tokens)
// A token: its gradient before its weight, KL term, ratio, the ratio that its loss takes, and whether that is a border's
struct PolicyToken { float g, kl, rho, used; bool cut; };

// e^x by the exponential unit, log2(e) in two parts: within (|x| + 2) 2^-24 of e^x, which the rounding of the difference x (|x| 2^-24)
// allows for.  Results below 2^-126 may be 0.
__device__ __forceinline__ float exp_near(float x) { return __builtin_amdgcn_exp2f(fmaf(x, 1.44269502f, x * 1.92596299e-8f)); }

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
    const float e = exp_near(x);
    m = e - 1.f;
    r = m - x;
  }
  *em1 = m;
  *rest = r;
}

// The KL term of x = ref - logp and its derivative by logp; KL 0: none, 1..3: the kinds
template <int KL>
__device__ __forceinline__ void kl_term(float x, float* kl, float* dk) {
  *kl = *dk = 0.f;
  if (KL == 1) { *kl = -x; *dk = 1.f; }
  if (KL == 2) { *kl = 0.5f * x * x; *dk = -x; }
  if (KL == 3) { float m; exp_parts(x, &m, kl); *dk = -m; }
}

// Is the token beyond a border (from the difference in float64), and the ratio that is held there
__device__ __forceinline__ bool beyond(const PolicyP& p, float lp, float old, float A, float* held) {
  const double x = (double)lp - (double)old;
  const float vhi = p.vhi, vlo = p.vlo, vdual = p.vdual;
  const bool over = A > 0.f && x > p.hi, far = A < 0.f && x > p.dual, under = A < 0.f && x < p.lo;
  *held = over ? vhi : (under ? vlo : vdual);
  return over || far || under;
}

template <int KL>
__device__ __forceinline__ PolicyToken policy_token(const PolicyP& p, float lp, float old, float ref, float A) {
  // (by value: a selection between fields of the kernel's arguments would be one of addresses, and put them into scratch)
  const float fhi = p.fhi, flo = p.flo, fdual = p.fdual, vhi = p.vhi, vlo = p.vlo, vdual = p.vdual;
  const float d = lp - old;
  float held = A > 0.f ? vhi : (d > 0.f ? vdual : vlo);
  PolicyToken q;
  q.cut = A > 0.f ? d > fhi : (A < 0.f && (d < flo || d > fdual));
  if (d == fhi || d == flo || d == fdual) q.cut = beyond(p, lp, old, A, &held);
  q.rho = exp_near(d);
  q.used = q.cut ? held : q.rho;
  q.g = q.cut ? 0.f : -A * q.rho;
  q.kl = 0.f;
  if (KL) {
    float dk;
    kl_term<KL>(ref - lp, &q.kl, &dk);
    q.g = fmaf(p.kl_coef, dk, q.g);
  }
  return q;
}
// A token's terms, u: 1 / its row's length
__device__ __forceinline__ void add_token(PolicySum& sum, const PolicyToken& q, float A, float u) {
  sum.pg = fma(-(double)A * (double)u, (double)q.used, sum.pg);
  sum.kl = fma((double)u, (double)q.kl, sum.kl);
  sum.rho += (double)q.rho;
}

// What multiplies a token besides 1 / (its row's length): 1 / tokens, 1 / sequences or 1 / denominator.
__device__ __forceinline__ double policy_weight(const PolicyP& p, double tokens, double rows) {
  if (p.fixed > 0.0) return p.fixed;
  const double n = p.mode == 0 ? tokens : rows;
  return n > 0.0 ? 1.0 / n : 0.0;
}
// ... from the partial counts, by every wave for itself, or (few rows, no mask) from the rows themselves
__device__ __forceinline__ double policy_weight_parts(const PolicyP& p, double* lds) {
  if (p.fixed > 0.0) return p.fixed;
  if (p.tk.packed && p.mode == 0 && !p.tk.mask) {     // the offsets say how many tokens there are
    const long long a = uniform_load(p.tk.cu), b = uniform_load(p.tk.cu + p.tk.rows), s = a < 0 ? 0 : a, e = b > p.tk.n ? p.tk.n : b;
    return policy_weight(p, (double)(e - s), 0.0);
  }
  double v[2] = {0, 0};
  if (p.nnp > 0) {
    static_assert(COUNT_BLOCKS <= 256, "four partial counts a lane");
    NormPart q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = (threadIdx.x & 63) + 64 * k;
      q[k] = NormPart{0, 0};
      if (i < p.nnp) q[k] = p.np[i];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[0] += (double)q[k].tokens;
      v[1] += (double)q[k].rows;
    }
    return policy_weight(p, wave_sum64(v[0]), wave_sum64(v[1]));
  }
#pragma unroll 8
  for (long long r = threadIdx.x; r < p.tk.rows; r += 256) {
    long long s, e;
    row_bounds(p.tk, r, &s, &e);
    v[0] += (double)(e - s);
    v[1] += e > s ? 1.0 : 0.0;
  }
  block_sum<2, 256>(v, lds);
  return policy_weight(p, v[0], v[1]);
}

// The last sequence that begins at or before token i (its first one is 0), searched in [lo, hi].
__device__ __forceinline__ int find_row(const int* cu, int lo, int hi, long long i) {
  while (lo < hi) {
    const int m = lo + ((hi - lo + 1) >> 1);
    if ((long long)cu[m] <= i) lo = m;
    else hi = m - 1;
  }
  return lo;
}
// The same for a token that is the same in the whole wave, by its 64 lanes (all of them active)
__device__ __forceinline__ int find_row_wave(const int* cu, int rows, long long i) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = rows;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int at = lane * step;
    const bool le = at < n && (long long)cu[lo + (at < n ? at : 0)] <= i;
    const int c = __popcll(__ballot(le));
    if (c == 0) return lo;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  return lo;
}

// What a row's tokens share
struct RowInfo { float A, u; };
__device__ __forceinline__ RowInfo row_info(const PolicyP& p, long long r, long long tokens) {
  RowInfo ri{p.acs ? 0.f : p.adv[r * p.ars], 1.f};
  if (p.mode == 1) {
    const long long c = p.counts ? (long long)p.counts[r] : tokens;
    ri.u = c > 0 ? 1.f / (float)c : 0.f;
  }
  return ri;
}

__device__ __forceinline__ long long row_of(const TokenP& t, long long i) {
  return t.n <= 0xffffffffll ? (long long)((unsigned)i / (unsigned)t.len) : i / t.len;
}

// Token i, whatever the views' strides and the rows' lengths; packed: its sequence is not before `first`
template <typename T>
__device__ __forceinline__ void policy_one(const PolicyP& p, long long i, float W, PolicySum& sum, int first = 0) {
  long long r, c, s, e;
  if (p.tk.packed) {
    r = find_row(p.tk.cu, first, (int)p.tk.rows - 1, i);
    c = i;
  } else {
    r = row_of(p.tk, i);
    c = i - r * p.tk.len;
  }
  row_bounds(p.tk, r, &s, &e);
  bool valid = c >= s && c < e;
  if (valid && p.tk.mask) valid = p.tk.mask[(p.tk.packed ? 0 : r * p.tk.mrs) + c * p.tk.mcs] != 0;
  float g = 0.f;
  if (valid) {
    const RowInfo ri = row_info(p, r, e - s);
    const long long k = p.tk.packed ? 0 : r;
    const float lp = load_one((const T*)p.lp + k * p.lrs + c * p.lcs);
    const float old = p.old ? load_one((const T*)p.old + k * p.ors + c * p.ocs) : lp;
    const float ref = p.ref ? load_one((const T*)p.ref + k * p.rrs + c * p.rcs) : 0.f;
    const float A = p.acs ? p.adv[k * p.ars + c * p.acs] : ri.A;
    const PolicyToken q = !p.ref ? policy_token<0>(p, lp, old, ref, A) : p.kl == 1 ? policy_token<1>(p, lp, old, ref, A)
                          : p.kl == 2 ? policy_token<2>(p, lp, old, ref, A) : policy_token<3>(p, lp, old, ref, A);
    g = q.g * (W * ri.u);
    add_token(sum, q, A, ri.u);
    sum.cut += q.cut;
    sum.cnt += 1;
  }
  if (p.grad) store_one((T*)p.grad + i, g);
}

template <typename T, int KL, bool TA, int N>
struct PolicyLoad {
  Pack<T, N> l, o, f;
  Pack<float, N> a;
  __device__ __forceinline__ void load(const PolicyP& p, long long i) {
    l.load((const T*)p.lp + i);
    o.load((const T*)(p.old ? p.old : p.lp) + i);
    if (KL) f.load((const T*)p.ref + i);
    if (TA) a.load(p.adv + i);
  }
};

// The rows of a thread's tokens i .. i + N - 1: the first k1 are of row a, the others of row b; bit e of valid: token i + e
// counts; single: more than two rows, looked up token by token; one_row: the whole wave lies in row a.  Packed: pos, the place
// of the first token's row in the wave's window (< 0: the window does not reach).
struct RowsOfPack { RowInfo a, b; int k1, pos; unsigned valid; bool single, one_row; };
__device__ __forceinline__ unsigned low_bits(int n) { return (1u << n) - 1u; }

// The begins of 64 sequences from `r` on, one a lane, kept from turn to turn: the tokens of a workgroup are consecutive, so
// most turns find their sequences without a load.
struct Window { int r, at; };

// All lanes active; iw .. lw: the wave's tokens
template <int N>
__device__ __forceinline__ RowsOfPack rows_packed(const PolicyP& p, Window& w, long long i, long long iw, long long lw) {
  const TokenP& t = p.tk;
  const int rows = (int)t.rows, lane = threadIdx.x & 63;
  RowsOfPack q;
  q.single = false;
  q.pos = -1;
  int k = 0;                                                           // the wave's first sequence is w.r + k
  if (w.r >= 0) k = max(0, __popcll(__ballot((long long)w.at <= iw)) - 1);
  if (w.r < 0 || k == 63 || (w.r + 61 < rows && (long long)__builtin_amdgcn_readlane(w.at, 61) <= lw)) {
    w.r = uniform(w.r < 0 || k == 63 ? find_row_wave(t.cu, rows, iw) : w.r + k);
    w.at = t.cu[min(w.r + lane, rows)];                                // (behind the last one: its end)
    k = 0;
  }
  k = uniform(k);
  const int o0 = __builtin_amdgcn_readlane(w.at, k), o1 = __builtin_amdgcn_readlane(w.at, k + 1), r = w.r + k;
  q.one_row = r < rows && o0 <= iw && lw < o1 && o1 <= t.n;
  if (q.one_row) {
    const long long c = p.counts && p.mode == 1 ? (long long)uniform_load(p.counts + r) : (long long)o1 - (o0 < 0 ? 0 : o0);
    q.a = q.b = RowInfo{p.acs ? 0.f : uniform_load(p.adv + r * p.ars), p.mode != 1 ? 1.f : c > 0 ? 1.f / (float)c : 0.f};
    q.k1 = N;
    q.valid = low_bits(N);
    return q;
  }
  if (w.r + 61 < rows && (long long)__builtin_amdgcn_readlane(w.at, 61) <= lw) {       // more sequences than lanes: the caller's policy_rest
    q.k1 = 0;
    q.valid = 0u;
    return q;
  }
  if (i >= t.n) i = t.n - 1;                                           // (a lane behind the end: its answer is not used)
  int pos = 0;
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
    if ((long long)__shfl(w.at, pos + step, 64) <= i) pos += step;
  pos = min(pos, min(rows - 1 - w.r, 61));
  q.pos = pos;
  const int row = w.r + pos;
  long long s = __shfl(w.at, pos, 64), e = __shfl(w.at, pos + 1, 64), e2 = __shfl(w.at, pos + 2, 64);
  s = s < 0 ? 0 : (s > t.n ? t.n : s);
  e = e < s ? s : (e > t.n ? t.n : e);
  e2 = e2 < e ? e : (e2 > t.n ? t.n : e2);
  const bool two = e < i + N && row + 1 < rows;
  q.single = i < s || (two && e2 < i + N && row + 2 < rows);
  q.k1 = e <= i ? 0 : e - i < N ? (int)(e - i) : N;
  q.a = q.b = row_info(p, row, e - s);
  int nb = 0;
  if (two) {
    nb = e2 >= i + N ? N - q.k1 : e2 <= i + q.k1 ? 0 : (int)(e2 - i) - q.k1;
    q.b = row_info(p, row + 1, e2 - e);
  }
  q.valid = low_bits(q.k1 + nb);
  return q;
}

template <int N>
__device__ __forceinline__ RowsOfPack rows_padded(const PolicyP& p, long long i, long long iw, long long lw) {
  const TokenP& t = p.tk;
  const long long L = t.len, r0 = uniform(row_of(t, iw));
  RowsOfPack q;
  q.single = false;
  q.pos = -1;
  q.one_row = lw < (r0 + 1) * L;
  long long s, e;
  if (q.one_row) {
    e = t.lengths ? (long long)uniform_load(t.lengths + r0) : L;
    e = e < 0 ? 0 : (e > L ? L : e);
    const long long c = i - r0 * L, m = p.mode != 1 ? 0 : p.counts ? (long long)uniform_load(p.counts + r0) : e;
    q.a = q.b = RowInfo{p.acs ? 0.f : uniform_load(p.adv + r0 * p.ars), p.mode != 1 ? 1.f : m > 0 ? 1.f / (float)m : 0.f};
    q.k1 = N;
    q.valid = low_bits(e <= c ? 0 : e - c < N ? (int)(e - c) : N);
    return q;
  }
  if (i >= t.n) i = t.n - 1;
  const long long r = row_of(t, i), c = i - r * L;
  row_bounds(t, r, &s, &e);
  q.k1 = L - c < N ? (int)(L - c) : N;
  q.valid = low_bits(e <= c ? 0 : e - c < q.k1 ? (int)(e - c) : q.k1);
  q.a = q.b = row_info(p, r, e);
  if (q.k1 < N && r + 1 < t.rows) {
    row_bounds(t, r + 1, &s, &e);
    q.valid |= low_bits(e < N - q.k1 ? (int)e : N - q.k1) << q.k1;
    q.b = row_info(p, r + 1, e);
  }
  return q;
}

// With s the advantage's sign a token is beyond the border where s d exceeds one number (and with a dual border where -s d,
// s < 0, exceeds another).
struct Border { float at, held; };
__device__ __forceinline__ Border border_of(const PolicyP& p, float A) {
  const float fhi = p.fhi, flo = p.flo, vhi = p.vhi, vlo = p.vlo;
  return {A > 0.f ? fhi : (A < 0.f ? -flo : INFINITY), A > 0.f ? vhi : vlo};
}
__device__ __forceinline__ float signed_by(float d, float A) { return __uint_as_float(__float_as_uint(d) ^ (__float_as_uint(A) & 0x80000000u)); }

// Does a rounded difference of the wave's tokens equal a border?
template <typename T, int KL, bool TA, int N, bool DUAL>
__device__ __forceinline__ bool at_border(const PolicyP& p, const PolicyLoad<T, KL, TA, N>& x, float rowA) {
  const float fdual = p.fdual;
  bool same = false;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float A = TA ? x.a.at(k) : rowA, d = x.l.at(k) - x.o.at(k);
    same = same || signed_by(d, A) == border_of(p, A).at || (DUAL && d == fdual);
  }
  return __any(same);
}

// N tokens of one row that all count, none of them at a border, in every lane: what the row shares is taken out of the sums.
template <typename T, int KL, bool TA, int N, bool DUAL>
__device__ __forceinline__ void policy_row(const PolicyP& p, const PolicyLoad<T, KL, TA, N>& x, RowInfo row, float W, float* g, PolicySum& sum) {
  const float w = W * row.u, wk = w * p.kl_coef, fdual = p.fdual, vdual = p.vdual;
  double used = 0.0, rhos = 0.0, kl = 0.0;
  unsigned cuts = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float A = TA ? x.a.at(k) : row.A;
    const Border b = border_of(p, A);
    const float l = x.l.at(k), d = l - x.o.at(k), rho = exp_near(d);
    bool cut = signed_by(d, A) > b.at;
    float r = cut ? b.held : rho, live = cut ? 0.f : rho;
    if (DUAL) {
      const bool far = A < 0.f && d > fdual;
      r = far ? vdual : r;
      live = far ? 0.f : live;
      cut = cut || far;
    }
    cuts += cut;
    rhos += (double)rho;
    if (TA) {
      used = fma(-(double)A, (double)r, used);
      g[k] = -A * live * w;
    } else {
      used += (double)r;
      g[k] = (-row.A * w) * live;
    }
    if (KL) {
      float q, dk;
      kl_term<KL>(x.f.at(k) - l, &q, &dk);
      kl += (double)q;
      g[k] = fmaf(wk, dk, g[k]);
    }
  }
  const double u = (double)row.u;
  sum.pg = fma(TA ? u : -(double)row.A * u, used, sum.pg);
  if (KL) sum.kl = fma(u, kl, sum.kl);
  sum.rho += rhos;
  sum.cut += cuts;
  sum.cnt += N;
}

// A thread's N tokens from i on, loaded into x, of the rows q; `mine`: they are all there.  All lanes active.
template <typename T, int KL, bool TA, bool PACKED, int N, bool DUAL>
__device__ __forceinline__ void policy_pack(const PolicyP& p, const Window& w, long long i, const PolicyLoad<T, KL, TA, N>& x, RowsOfPack q,
                                            unsigned masked, bool mine, float W, PolicySum& sum) {
  float g[N];
  const bool row = __all(q.valid == low_bits(N)) && q.one_row && !at_border<T, KL, TA, N, DUAL>(p, x, q.a.A);
  auto token = [&](int k, bool on, float A, float u) {     // where tokens may not count: their values are replaced, their e^0 is left out
    const float l = on ? x.l.at(k) : 0.f, o = on ? x.o.at(k) : 0.f, f = KL && on ? x.f.at(k) : 0.f;
    const float t = TA ? x.a.at(k) : A, At = on ? t : 0.f, ut = on ? u : 0.f;
    PolicyToken v = policy_token<KL>(p, l, o, f, At);
    v.rho = on ? v.rho : 0.f;
    add_token(sum, v, At, ut);
    sum.cut += on && v.cut;
    sum.cnt += on;
    g[k] = on ? W * ut * v.g : 0.f;
    // one token after the other: all of them side by side do not fit the registers (scratch in every 16-bit kernel)
    asm volatile("" : "+v"(sum.pg), "+v"(sum.kl), "+v"(sum.rho), "+v"(g[k]));
  };
  if (row) {
    policy_row<T, KL, TA, N, DUAL>(p, x, q.a, W, g, sum);
  } else if (PACKED && !q.one_row && __any(q.single)) {    // some lane's tokens lie in more than two sequences: all look each token up
    int pos = q.pos;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      for (;;) {                                      // past the sequences that end here (empty ones too)
        const long long next = __shfl(w.at, pos + 1, 64);                // (by all lanes: a lane that sat out could not be read)
        const bool on = pos < 62 && w.r + pos + 1 < p.tk.rows && next <= i + k;
        if (!__any(on)) break;
        pos += on;
      }
      long long s = __shfl(w.at, pos, 64), e = __shfl(w.at, pos + 1, 64);
      s = s < 0 ? 0 : (s > p.tk.n ? p.tk.n : s);
      e = e < s ? s : (e > p.tk.n ? p.tk.n : e);
      const RowInfo ri = row_info(p, w.r + pos, e - s);
      token(k, mine && i + k >= s && i + k < e && (masked & (1u << k)), ri.A, ri.u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) token(k, (q.valid >> k) & 1u, k < q.k1 ? q.a.A : q.b.A, k < q.k1 ? q.a.u : q.b.u);
  }
  if (p.grad && mine) store_vec<N>((T*)p.grad + i, g);
}

// A wave's tokens behind the last whole N, one a lane; or, more sequences than its window takes, all of them one by one
template <typename T, int N>
__device__ __forceinline__ void policy_rest(const PolicyP& p, const Window& w, bool all, long long i, long long iw, long long lw, float W,
                                            PolicySum& sum) {
  const int first = w.r < 0 ? 0 : w.r;
  if (all) {
    for (int k = 0; k < N; ++k)
      if (i + k <= lw) policy_one<T>(p, i + k, W, sum, first);
    return;
  }
  const long long t = iw + (lw + 1 - iw) / N * N + (threadIdx.x & 63);
  if (t <= lw) policy_one<T>(p, t, W, sum, first);
}

// Tokens [begin, end) of flat tensors by a workgroup.  Where a mask or lengths say which tokens count, the loads wait for
// that (p.early: not in calls of one turn, which latency bounds).
template <typename T, int KL, bool TA, bool PACKED, bool DUAL>
__device__ __forceinline__ void policy_flat(const PolicyP& p, long long begin, long long end, float W, PolicySum& sum) {
  constexpr int N = 16 / (int)sizeof(T);
  Window win{-1, 0};
  for (long long b = begin; b < end; b += 256 * N) {
    const long long i = b + threadIdx.x * N, iw = uniform(b + (threadIdx.x & ~63) * N);
    if (iw >= end) break;
    const long long lw = iw + 64 * N <= end ? iw + 64 * N - 1 : end - 1;
    const bool whole = i + N <= end;
    PolicyLoad<T, KL, TA, N> x;
    typedef unsigned char bytes __attribute__((ext_vector_type(N), aligned(1)));
    bytes m;
    if (p.tk.mask && whole) m = *(const TREBI_GLOBAL bytes*)(p.tk.mask + i);
    if (p.early && whole) x.load(p, i);
    RowsOfPack q = PACKED ? rows_packed<N>(p, win, i, iw, lw) : rows_padded<N>(p, i, iw, lw);
    unsigned masked = low_bits(N);
    if (p.tk.mask) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (!m[k]) masked &= ~(1u << k);
    }
    q.valid &= whole ? masked : 0u;
    q.single = q.single && whole;
    if (PACKED && !q.one_row && q.pos < 0) {
      policy_rest<T, N>(p, win, true, i, iw, lw, W, sum);
      continue;
    }
    if (!p.early && (q.valid || q.single)) x.load(p, i);
    if (__any(q.valid || q.single)) {
      policy_pack<T, KL, TA, PACKED, N, DUAL>(p, win, i, x, q, masked, whole, W, sum);
    } else if (p.grad && whole) {                     // a wave of tokens that do not count
      const float zero[N] = {};
      store_vec<N>((T*)p.grad + i, zero);
    }
    if ((lw + 1 - iw) % N) policy_rest<T, N>(p, win, false, i, iw, lw, W, sum);
  }
}

// The same for packed sequences without a mask: the loads of a turn go out before the turn before it is computed, and
// without a condition (past the end: the last tokens again), so that nothing waits for them but their own use.
template <typename T, int KL, bool TA, bool DUAL>
__device__ __forceinline__ void policy_stream(const PolicyP& p, long long begin, long long end, float W, PolicySum& sum) {
  constexpr int N = 16 / (int)sizeof(T);
  Window win{-1, 0};
  PolicyLoad<T, KL, TA, N> x, next;
  const long long last = p.tk.n - N, mine = threadIdx.x * N;
  x.load(p, min(begin + mine, last));
  for (long long b = begin; b < end; b += 256 * N) {
    const long long i = b + mine, iw = uniform(b + (threadIdx.x & ~63) * N);
    next.load(p, min(b + 256 * N < end ? i + 256 * N : i, last));
    if (iw < end) {
      const long long lw = iw + 64 * N <= end ? iw + 64 * N - 1 : end - 1;
      RowsOfPack q = rows_packed<N>(p, win, i, iw, lw);
      const bool whole = i + N <= end;
      if (q.one_row || q.pos >= 0) {
        if (!whole) q.valid = 0u;
        q.single = q.single && whole;
        policy_pack<T, KL, TA, true, N, DUAL>(p, win, i, x, q, low_bits(N), whole, W, sum);
        if ((lw + 1 - iw) % N) policy_rest<T, N>(p, win, false, i, iw, lw, W, sum);
      } else {
        policy_rest<T, N>(p, win, true, i, iw, lw, W, sum);
      }
    }
    x = next;
  }
}

// KIND 0: any strides, token by token; 1: flat padded rows; 2: packed; 3: packed with a mask.  DUAL: is there a dual border (decided
// inside the kernel it costs the registers of both).  Waves on a SIMD: 5 where that pays (4096 x 8192 bfloat16, second KL term: 63 us,
// with 4: 76), 4 for the others (packed, masked, bfloat16, third KL term, an advantage a token: 28 us, with 5: 31; 512 x 2047: 14.8 and
// 15.1).  No instance spills vector registers.
template <typename T, int KL, bool TA, int KIND, bool DUAL>
__global__ __launch_bounds__(256, KIND == 1 && !TA && KL < 3 ? 5 : 4) void policy_kernel(PolicyP p) {
  __shared__ double lds[5 * LOSS_VALS];
  const double W = policy_weight_parts(p, lds);
  const float Wg = (float)(W * (double)p.gscale);
  const long long begin = (long long)blockIdx.x * p.per, end = begin + p.per < p.tk.n ? begin + p.per : p.tk.n;
  PolicySum sum{0, 0, 0, 0, 0};
  if (KIND == 0) {
    for (long long i = begin + threadIdx.x; i < end; i += 256) policy_one<T>(p, i, Wg, sum);
  } else {
    if constexpr (KIND == 2) policy_stream<T, KL, TA, DUAL>(p, begin, end, Wg, sum);
    else policy_flat<T, KL, TA, KIND == 3, DUAL>(p, begin, end, Wg, sum);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && gridDim.x > 1) *p.weight = W;
  double acc[LOSS_VALS] = {sum.pg, sum.kl, (double)sum.cut, sum.rho, (double)sum.cnt};
  block_sum<LOSS_VALS, 256>(acc, lds);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) policy_stats(p, acc, W);
    else
#pragma unroll
      for (int k = 0; k < LOSS_VALS; ++k) p.part[k * LOSS_PARTS + blockIdx.x] = acc[k];
  }
}

template <typename T, int KL>
static hipError_t launch_policy_k(const PolicyP& p, int blocks, hipStream_t st) {
#define GO(TA, KIND)                                                                                                              \
  do {                                                                                                                            \
    if (p.dual < INFINITY) hipLaunchKernelGGL((policy_kernel<T, KL, TA, KIND, true>), dim3(blocks), dim3(256), 0, st, p);         \
    else hipLaunchKernelGGL((policy_kernel<T, KL, TA, KIND, false>), dim3(blocks), dim3(256), 0, st, p);                          \
  } while (0)
  if (!p.tk.packed) { if (p.acs) GO(true, 1); else GO(false, 1); }
  else if (!p.tk.mask) { if (p.acs) GO(true, 2); else GO(false, 2); }
  else { if (p.acs) GO(true, 3); else GO(false, 3); }
  return hipGetLastError();
}
template <typename T>
static hipError_t launch_policy_t(const PolicyP& p, int blocks, hipStream_t st) {
  if (!p.flat) {
    hipLaunchKernelGGL((policy_kernel<T, 0, false, 0, true>), dim3(blocks), dim3(256), 0, st, p);
    return hipGetLastError();
  }
  switch (p.ref ? p.kl : 0) {
    case 0: return launch_policy_k<T, 0>(p, blocks, st);
    case 1: return launch_policy_k<T, 1>(p, blocks, st);
    case 2: return launch_policy_k<T, 2>(p, blocks, st);
    default: return launch_policy_k<T, 3>(p, blocks, st);
  }
#undef GO
}

}  // namespace trebi
