"""GPU: how exact the fine-tuning losses are where errors do not average out: sums of many equal terms, means over few tokens among
many that do not count, tokens exactly at a border, pairs far from the middle."""
import math

import numpy as np
import pytest
import torch

import _finetune as F
from test_gpu_losses import DT, ULP, check_policy, np64, rows_of

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------- few valid tokens
@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('layout', ['mask', 'lengths', 'packed'])
def test_mean_ratio_of_few_small_ratios(layout, dtype):
    """Rows of 512 tokens of which one in eight (mask) or the first three (lengths, packed behind a long row) count, all at a
    ratio of e^-8: the mean is that ratio, within an exponential's error ((1.25 * 8 + 2) 2^-24) and a rounding: ULP of it."""
    from trebi_amd.losses import policy_loss
    R, L = 16, 512
    lp, old = torch.full((R, L), -9.0), torch.full((R, L), -1.0)
    kw = {}
    if layout == 'mask':
        keep = torch.zeros(R, L, dtype=torch.bool)
        keep[:, 5::8] = True
        kw['mask'] = keep.cuda()
    else:
        kw['lengths'] = torch.full((R,), 3).cuda()
    lp, old = lp.to(DT[dtype]).cuda(), old.to(DT[dtype]).cuda()
    if layout == 'packed':
        n = R * L
        kw = dict(cu_seqlens=torch.tensor([7 * k for k in range(R)] + [7 * R], device='cuda').clamp(max=n),
                  mask=(torch.arange(n, device='cuda') % 7 < 3))
        lp, old = lp.reshape(-1), old.reshape(-1)
    adv = torch.ones(R, device='cuda')
    r = policy_loss(lp, adv, old, **kw)
    assert abs(float(r.ratio) - math.exp(-8)) <= ULP * math.exp(-8)
    assert abs(float(r.loss) + math.exp(-8)) <= ULP * math.exp(-8)


# ------------------------------------------------------------------------------------------------- equal terms
LAYOUTS = ['all', 'lengths', 'mask', 'packed', 'packed-mask']


def equal_layout(layout, R, L):
    """(shape, which=, number of valid tokens of each row)"""
    rng = np.random.default_rng(0)
    if layout == 'all':
        return (R, L), {}, np.full(R, L)
    n = np.arange(R) * (L // R) + 1
    if layout == 'lengths':
        return (R, L), dict(lengths=torch.from_numpy(n).cuda()), n
    if layout == 'mask':
        m = rng.random((R, L)) < 0.7
        return (R, L), dict(mask=torch.from_numpy(m).cuda()), m.sum(1)
    cu = np.concatenate([[0], np.cumsum(n * 8)])
    kw = dict(cu_seqlens=torch.from_numpy(cu).cuda())
    if layout == 'packed':
        return (int(cu[-1]),), kw, n * 8
    m = rng.random(cu[-1]) < 0.7
    return (int(cu[-1]),), dict(mask=torch.from_numpy(m).cuda(), **kw), np.array([m[a:b].sum() for a, b in zip(cu, cu[1:])])


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('layout', LAYOUTS)
def test_policy_sums_of_one_advantage_a_token_have_no_bias(layout, dtype):
    """Every token held at its border, with advantages +1 and -1 given for each token, the same over runs of 512: each term is one of two
    float32 numbers (1.28 and 0.8 as float32), and a sum in float64 leaves only the result's own rounding."""
    from trebi_amd.losses import policy_loss
    shape, which, _ = equal_layout(layout, 64, 1024)
    sign = torch.where(torch.arange(int(np.prod(shape))) // 512 % 2 == 0, 1.0, -1.0).reshape(shape)
    old = torch.full(shape, -1.0)
    logp = old + 0.5 * sign
    r = policy_loss(logp.to(DT[dtype]).cuda(), sign.cuda(), old.to(DT[dtype]).cuda(), clip=0.2, clip_high=0.28, per_token=True, **which)
    valid = torch.ones(shape, dtype=torch.bool)
    if 'lengths' in which:
        valid = torch.arange(shape[1])[None] < which['lengths'].cpu()[:, None]
    if 'mask' in which:
        valid = which['mask'].cpu()
    hi, lo = float(np.float32(1 + float(np.float32(0.28)))), float(np.float32(1 - float(np.float32(0.2))))
    up, n = int((valid & (sign > 0)).sum()), int(valid.sum())
    want = (-hi * up + lo * (n - up)) / n
    assert float(r.clip_fraction) == 1.0
    assert abs(float(r.policy) - want) <= F.F24 * abs(want) + 2.0 ** -50


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('adv', ['row', 'token'])
def test_mean_ratio_and_kl_of_equal_tokens_are_the_token_s(layout, dtype, adv):
    """N equal terms v: the float64 sum is N v exactly (N < 2^29), its mean v, and float32(v) the value of a single token's call.
    (No additions are fused differently by a compiler in these terms: each is a product or one difference.)"""
    from trebi_amd.losses import policy_loss
    shape, which, _ = equal_layout(layout, 32, 1024)
    for kl, lp, old, ref in (('k1', -1.125, -1.375, -1.6875), ('k2', -0.3125, -0.375, -0.7421875), ('k3', -1.15625, -1.3125, -1.4375)):
        v = [torch.full(shape, x).to(DT[dtype]).cuda() for x in (lp, old, ref)]
        A = torch.full(shape if adv == 'token' else (32,), 0.5, device='cuda')
        r = policy_loss(v[0], A, v[1], v[2], kl=kl, kl_coef=0.1, clip=0.5, per_token=adv == 'token', **which)
        one = [x.reshape(-1)[:1] for x in v]
        s = policy_loss(one[0], A.reshape(-1)[:1], one[1], one[2], kl=kl, kl_coef=0.1, clip=0.5)
        assert float(r.ratio) == float(s.ratio) and float(r.kl) == float(s.kl), (kl, float(r.kl), float(s.kl))
        assert abs(float(r.ratio) - math.exp(lp - old)) <= ULP * math.exp(lp - old)


# ------------------------------------------------------------------------------------------------- exactly at a border
@pytest.mark.parametrize('adv', ['row', 'token'])
@pytest.mark.parametrize('layout', ['all', 'packed'])
@pytest.mark.parametrize('dual', [None, 3.0])
def test_single_tokens_at_each_border_of_whole_rows(layout, adv, dual):
    """Rows of 2048 valid tokens, so that whole waves take one row: in each row one token has the float32 value of a border, or the
    value next to it on either side.  Which side a token is on follows from its value in float64."""
    from trebi_amd.losses import policy_loss
    lo32, hi32 = float(np.float32(0.2)), float(np.float32(0.28))
    borders = [math.log1p(hi32), math.log1p(-lo32), math.log(3.0)]
    vals = []
    for b in borders:
        v = np.float32(b)
        vals += [v, np.nextafter(v, np.float32(-9)), np.nextafter(v, np.float32(9))]
    L, rng = 2048, np.random.default_rng(3)
    R = 2 * len(vals)                                       # each value with advantages of both signs
    lp = (0.02 * rng.standard_normal((R, L))).astype(np.float32)
    A = np.repeat([1.5, -0.75], len(vals)).astype(np.float32)
    at = rng.integers(0, L, size=R)
    for r in range(R):
        lp[r, at[r]] = vals[r % len(vals)]
    At = np.repeat(A[:, None], L, 1)
    if adv == 'token':
        other = rng.random((R, L)) < 0.5
        other[np.arange(R), at] = False
        At = np.where(other, -At, At).astype(np.float32)
    old = np.zeros_like(lp)
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    flat = (lambda v: v.reshape(-1)) if layout == 'packed' else (lambda v: v)
    kw = dict(cu_seqlens=torch.arange(R + 1, device='cuda') * L) if layout == 'packed' else {}
    got = policy_loss(cu(flat(lp)), cu(flat(At)) if adv == 'token' else cu(A), cu(flat(old)), clip=0.2, clip_high=0.28, dual_clip=dual, **kw)
    want = F.policy(list(lp.astype(np.float64)), list(At.astype(np.float64)), list(old.astype(np.float64)), None, clip=lo32, clip_high=hi32, dual=dual)
    picks = [np.arange(L) + (r * L if layout == 'packed' else 0) for r in range(R)]
    check_policy(got, want, picks, 'float32', dict(abs_pg=1.5 * 3, abs_kl=1.0), (layout, adv, dual))
    g = np64(got.grad).reshape(R, L)[np.arange(R), at]
    wg = np.array([want[5][r][at[r]] for r in range(R)])
    assert ((g == 0) == (wg == 0)).all()


# ------------------------------------------------------------------------------------------------- far from the middle
def test_preference_loss_and_slope_of_decided_pairs():
    """The loss of a pair z > 0 apart is log(1 + e^-z) and its slope -sigmoid(-z): small numbers, right to the float32 they are
    returned in (everything before is float64; two roundings allowed), where z itself is not a float32 number too."""
    from trebi_amd.losses import preference_loss
    for margin in (0.0, 0.1, 1e-7):
        for c, r in ((0.0, -2.0), (-1.0, -6.1), (0.0, -20.0), (-0.3, -40.7), (-3.0, -83.0), (-20.0, -0.7), (-80.3, -1.0)):
            lp = torch.tensor([[c], [r]])
            z = float(lp[0, 0]) - float(lp[1, 0]) - float(np.float32(margin))
            got = preference_loss(lp.cuda(), beta=1.0, margin=margin)
            loss = math.log1p(math.exp(-abs(z))) + max(-z, 0.0)
            slope = 1 / (1 + math.exp(z))
            assert abs(float(got.loss) - loss) <= 2 * F.F24 * loss, (c, r, margin)
            assert abs(float(got.grad[0, 0]) + slope) <= 2 * F.F24 * slope and abs(float(got.grad[1, 0]) - slope) <= 2 * F.F24 * slope, (c, r, margin)
            e = float(np.float32(0.1))
            got = preference_loss(lp.cuda(), beta=1.0, margin=margin, label_smoothing=0.1)
            other = math.log1p(math.exp(-abs(z))) + max(z, 0.0)
            loss, sl = (1 - e) * loss + e * other, e / (1 + math.exp(-z)) - (1 - e) * slope
            assert abs(float(got.loss) - loss) <= 2 * F.F24 * loss
            assert abs(float(got.grad[0, 0]) - sl) <= 2 * F.F24 * abs(sl) + 2.0 ** -50


# ------------------------------------------------------------------------------------------------- the ratio itself
@pytest.mark.parametrize('adv', ['row', 'token'])
def test_every_ratio_is_within_its_bound(adv):
    """With advantages of -+1, weight 1 and no old log-probability but 0, a token's gradient is +- its ratio, unrounded: e^x within
    (|x| + 2) 2^-24 (the exponential's argument rounded in base 2, one step of the exponential unit).  Arguments just above a power
    of two in base 2, where that rounding is largest."""
    from trebi_amd.losses import policy_loss
    rng = np.random.default_rng(0)
    L = 8192
    for k in range(-1, 7):
        x = (math.log(2) * 2.0 ** k * (1 + 0.06 * rng.random((2, L)))).astype(np.float32)
        x[1] *= -1
        A = torch.tensor([-1.0, 1.0], device='cuda')            # no border holds ratios above 1 here, nor those below 1 there
        lp = torch.from_numpy(x).cuda()
        r = policy_loss(lp, A if adv == 'row' else A[:, None].expand(2, L).contiguous(), torch.zeros_like(lp), denominator=1.0)
        got, want = np.abs(np64(r.grad)), np.exp(x.astype(np.float64))
        assert float(r.clip_fraction) == 0.0
        assert (np.abs(got / want - 1) <= (np.abs(x) + 2) * F.F24).all(), (k, np.abs(got / want - 1).max() / F.F24)
