"""The fine-tuning operators' definitions in float64 numpy, token by token -- what the GPU tests hold the kernels to.
Inputs are the tensors' own (already rounded) values."""
import math

import numpy as np

F24 = 2.0 ** -24                 # half a unit in the last place of float32, relative
HALF = {'float32': 2.0 ** -24, 'bfloat16': 2.0 ** -8, 'float16': 2.0 ** -11}      # a rounding to the type, relative
TINY = {'float32': 2.0 ** -149, 'bfloat16': 2.0 ** -133, 'float16': 2.0 ** -24}   # the type's smallest step


def policy(rows, adv, old=None, ref=None, clip=0.2, clip_high=None, dual=None, coef=0.0, kl='k3', reduction='token',
           denominator=None):
    """rows: list of float64 arrays (a row's valid tokens); adv / old / ref likewise.  Returns (loss, policy, kl, share cut, mean
    ratio, gradients, magnitudes): a magnitude is the sum of the absolute terms of a gradient, what rounding errors scale with."""
    clip_high = clip if clip_high is None else clip_high
    N, S = sum(len(r) for r in rows), sum(len(r) > 0 for r in rows)
    pg_s = kl_s = cut_n = rho_s = 0.0
    grads, mags = [], []
    for i, r in enumerate(rows):
        g, m = np.zeros(len(r)), np.zeros(len(r))
        for j in range(len(r)):
            w = 1 / denominator if denominator else 1 / N if reduction == 'token' else 1 / (S * len(r))
            A = adv[i][j]
            d = r[j] - old[i][j] if old is not None else r[j] - r[j]
            with np.errstate(over='ignore', invalid='ignore'):
                rho = float(np.exp(d))
            held = None
            if A > 0 and d > math.log1p(clip_high):
                held = 1 + clip_high
            elif A < 0 and clip < 1 and d < math.log1p(-clip):
                held = 1 - clip
            elif A < 0 and dual and d > math.log(dual):
                held = dual
            with np.errstate(over='ignore', invalid='ignore'):
                pg = -A * (rho if held is None else held)
            dpg = pg if held is None else 0.0
            k = dk = 0.0
            if ref is not None:
                x = ref[i][j] - r[j]
                with np.errstate(over='ignore', invalid='ignore'):
                    e = float(np.expm1(x))
                k, dk = {'k1': (-x, 1.0), 'k2': (x * x / 2, -x), 'k3': (e - x, -e)}[kl]
            pg_s += w * pg
            kl_s += w * k
            cut_n += held is not None
            rho_s += rho
            g[j], m[j] = w * (dpg + coef * dk), w * (abs(dpg) + abs(coef * dk))
        grads.append(g)
        mags.append(m)
    return pg_s + coef * kl_s, pg_s, kl_s, cut_n / max(N, 1), rho_s / max(N, 1), grads, mags


def preference(rows, ref=None, weights=None, beta=0.1, kind='sigmoid', smooth=0.0, margin=0.0, average=False, denominator=None):
    """rows: 2 P lists of valid tokens.  (loss, rewards of the chosen, of the rejected, accuracy, mean z, gradient of each row's
    tokens, magnitude of the rows' sums)."""
    P = len(rows) // 2
    D, n = [], [len(r) for r in rows]
    for i, r in enumerate(rows):
        s = float(np.sum(r)) - (float(np.sum(ref[i])) if ref is not None else 0.0)
        D.append(s / n[i] if average and n[i] else s)
    loss = acc = zs = 0.0
    m = 0
    g = [0.0] * (2 * P)
    for k in range(P):
        if not n[k] or not n[k + P]:
            continue
        h = D[k] - D[k + P]
        z = beta * h - margin
        soft = lambda v: max(v, 0.0) + math.log1p(math.exp(-abs(v)))
        sig = lambda v: 1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v))
        if kind == 'sigmoid':
            one, slope = (1 - smooth) * soft(-z) + smooth * soft(z), beta * (smooth * sig(z) - (1 - smooth) * sig(-z))
        elif kind == 'hinge':
            one, slope = max(0.0, 1 - z), -beta if z < 1 else 0.0
        else:
            a = z / beta - 1 / (2 * beta)
            one, slope = a * a, 2 * a
        w = 1.0 if weights is None else float(weights[k])
        d = denominator or P
        loss += w * one / d
        slope *= w / d
        g[k], g[k + P] = slope / (n[k] if average else 1), -slope / (n[k + P] if average else 1)
        acc, zs, m = acc + (h > 0), zs + z, m + 1
    return loss, np.array([beta * v for v in D[:P]]), np.array([beta * v for v in D[P:]]), acc / max(m, 1), zs / max(m, 1), g


def schedule(T):
    """The cosine schedule's tables, float32 values as the planner holds them."""
    import torch
    from trebi_amd.diffusion import GaussianDiffusion
    import torch.nn as nn
    m = GaussianDiffusion(nn.Identity(), 4, 2, 1, n_timesteps=T, predict_epsilon=False)
    return {k: v.double().numpy() for k, v in m.named_buffers() if v.shape == (T,)}


def transition(tabs, pred, x, xp, t, act, obs, cond, epsilon, clamp):
    """(logp [B], d logp / d pred [B, H, D], sum of the absolute terms [B])"""
    B, H, D = pred.shape
    lp, g, mag = np.zeros(B), np.zeros((B, H, D)), np.zeros(B)
    free = np.ones((H, D), bool)
    for h in cond:
        free[h, act:act + obs] = False
    for b in range(B):
        k = int(t[b])
        if k == 0:
            continue
        raw = pred[b]
        c = 1.0
        if epsilon:
            raw = tabs['sqrt_recip_alphas_cumprod'][k] * x[b] - tabs['sqrt_recipm1_alphas_cumprod'][k] * pred[b]
            c = -tabs['sqrt_recipm1_alphas_cumprod'][k]
        x0 = np.clip(raw, -1, 1) if clamp else raw
        live = (np.abs(raw) <= 1) if clamp else np.ones_like(raw, bool)
        mu = tabs['posterior_mean_coef1'][k] * x0 + tabs['posterior_mean_coef2'][k] * x[b]
        plv = tabs['posterior_log_variance_clipped'][k]
        r = xp[b] - mu
        terms = -r * r / (2 * np.exp(plv)) - 0.5 * (np.log(2 * np.pi) + plv)
        lp[b], mag[b] = terms[free].sum(), np.abs(terms[free]).sum()
        g[b] = np.where(free & live, r / np.exp(plv) * tabs['posterior_mean_coef1'][k] * c, 0.0)
    return lp, g, mag
