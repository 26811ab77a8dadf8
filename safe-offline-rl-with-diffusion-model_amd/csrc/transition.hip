// Log-probability of a denoise transition, and its gradient with respect to the net's output.
#include "finetune.h"
#include "tokens.h"

namespace trebi {

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
// A wave (or a workgroup, where candidates are large or few) takes a candidate, so its timestep and table rows come
// through the scalar cache while its first elements are already on their way.  Bound by memory from some thousand candidates
// on: 32768 of 32 x 23 backwards, 386 MB, 71 us (5.4 TB/s: a part is read from the caches); below by the launch: 64 candidates, 3.7 us.
template <bool BWD, int G>
__global__ __launch_bounds__(256) void transition_kernel(TransP p) {
  __shared__ double lds[5];
  const int lane = threadIdx.x & (G - 1), per = 256 / G;
  const int n = p.H * p.D;
  typedef typename Vec<float, 4>::type vec;
  for (long long b0 = (long long)blockIdx.x * per; b0 < p.B; b0 += (long long)gridDim.x * per) {
    const long long b = uniform(b0 + threadIdx.x / G);
    const bool on = b < p.B;
    double acc = 0, plv = 0;
    long long tt = 0;
    if (on) {
      const float *pr = p.pred + b * p.prs, *xt = p.x + b * p.xrs, *xp = p.xp + b * p.xprs;
      vec vp = {0, 0, 0, 0}, vx = {0, 0, 0, 0}, vq = {0, 0, 0, 0};
      auto fetch = [&](int i) {
        if (i + 4 <= n) {
          vp = *(const TREBI_GLOBAL vec*)(pr + i);
          vx = *(const TREBI_GLOBAL vec*)(xt + i);
          vq = *(const TREBI_GLOBAL vec*)(xp + i);
        } else {
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (i + e < n) {
              vp[e] = load_one(pr + i + e);
              vx[e] = load_one(xt + i + e);
              vq[e] = load_one(xp + i + e);
            }
        }
      };
      fetch(lane * 4);
      tt = uniform_load(p.t + b);
      tt = tt < 0 ? 0 : (tt >= p.T ? p.T - 1 : tt);
      plv = (double)uniform_load(p.plv + tt);
      const double c1 = (double)uniform_load(p.c1 + tt), c2 = (double)uniform_load(p.c2 + tt);
      const double ra = p.ra ? (double)uniform_load(p.ra + tt) : 0.0, rm = p.ra ? (double)uniform_load(p.rm + tt) : 0.0;
      const double slope = BWD ? (double)uniform_load(p.g + b) * exp(-plv) * c1 * (p.ra ? -rm : 1.0) : 0.0;
      float* o = BWD ? p.dpred + b * (long long)n : nullptr;
      for (int i = lane * 4; i < n; i += G * 4) {
        const int m = n - i < 4 ? n - i : 4;
        float d[4] = {0, 0, 0, 0};
        if (tt > 0) {
          if (i > lane * 4) fetch(i);
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
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (e < m) store_one(o + i + e, d[e]);
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
      if (lane == 0 && on)
        p.logp[b] = tt > 0 ? (float)(-0.5 * acc * exp(-plv) - p.half_const * (1.8378770664093454836 + plv)) : 0.f;
    }
  }
}
hipError_t launch_transition(const TransP& p, int backward, hipStream_t st) {
  // A workgroup a candidate where a wave would go over its elements more than 16 times, or where there are so few
  // candidates that what one wave goes through is what the call takes.  32 x 23 elements, forwards: 64 candidates 3.7 us, a wave
  // each 5.1; 1024: 4.6 and 5.6; 2048: 8.1 and 7.0.  400 x 23: 64 candidates 10 and 34 us, 16384 289 and 297.  8 x 5: 1024 4.2 and 3.7.
  const long long n = (long long)p.H * p.D;
  const bool wide = n > 4096 || (p.B <= 1024 && n > 256);
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
