"""GPU: the policy loss, the preference loss and the transition log-probability against their definitions in float64
(tests/_finetune.py), at the sizes, masks, strides and types where such kernels go wrong.

Tolerances.  A gradient element is a product of fewer than 8 float32 factors, one of them an exponential (within (|x| + 2) 2^-24 of
its value) of an argument x rounded to float32 (relative 2^-24, so the exponential moves by |x| 2^-24): with |x| <= 8 that is at
most (8 + 10 + 8) * 2^-24 of the sum of the terms' magnitudes; 32 * 2^-24 is allowed, plus one rounding to the
output's type (HALF of the value, and TINY, its smallest step).  Scalars are float64 sums of such terms, rounded to float32:
32 * 2^-24 of the sum of the terms' magnitudes."""
import math

import numpy as np
import pytest
import torch

import _finetune as F

pytestmark = pytest.mark.gpu
DT = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
ULP = 32 * F.F24


def np64(v):
    return v.detach().cpu().double().numpy()


def rand(g, *shape, dtype='float32', scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(DT[dtype])


def build(layout, rows, length, seed, dtype='float32', scale=0.6):
    """(tensors maker, which=, picks): picks[r] = index of row r's valid tokens."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    if layout.startswith('packed'):
        lens = rng.integers(0, 2 * length + 1, size=rows)
        if rows > 2:
            lens[rows // 2] = 0
        front, tail = (3, 5) if layout != 'packed-tight' else (0, 0)
        cu = np.concatenate([[0], np.cumsum(lens)]) + front
        n = int(cu[-1]) + tail
        shape, which = (n,), dict(cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda())
        picks = [np.arange(cu[r], cu[r + 1]) for r in range(rows)]
        if layout == 'packed-mask':
            m = rng.random(n) < 0.6
            which['mask'] = torch.from_numpy(m).cuda()
            picks = [p[m[p]] for p in picks]
        return g, shape, which, picks
    shape, which = (rows, length), {}
    ok = np.ones(shape, bool)
    if 'lengths' in layout:
        lens = rng.integers(0, length + 1, size=rows)
        if rows > 1:
            lens[0] = 0                                     # a row that is all padding
        which['lengths'] = torch.from_numpy(lens).cuda()
        ok &= np.arange(length)[None] < lens[:, None]
    if 'mask' in layout:
        m = rng.random(shape) < 0.6
        if rows > 1:
            m[rows - 1] = False                             # a row whose mask leaves nothing
        which['mask'] = torch.from_numpy(m).cuda()
        ok &= m
    return g, shape, which, [np.nonzero(ok[r])[0] for r in range(rows)]


def rows_of(v, picks):
    v = np64(v)
    return [v[p] if v.ndim == 1 else v[r][p] for r, p in enumerate(picks)]


def unpack(v, picks):
    """Values at valid tokens in row order, and the largest magnitude elsewhere."""
    v = np64(v)
    out, rest = [], v.copy()
    for r, p in enumerate(picks):
        row = v if v.ndim == 1 else v[r]
        out.append(row[p])
        (rest if v.ndim == 1 else rest[r])[p] = 0.0
    return out, float(np.abs(rest).max()) if rest.size else 0.0


def check_policy(r, want, picks, dtype, kw, where=''):
    loss, pg, kl, cut, ratio, grads, mags = want
    got, rest = unpack(r.grad, picks)
    assert rest == 0.0, where
    for i, (a, b, m) in enumerate(zip(got, grads, mags)):
        err = np.abs(a - b)
        assert (err <= ULP * m + F.HALF[dtype] * np.abs(b) + F.TINY[dtype]).all(), (where, i, float(err.max()))
    total = sum(float(m.sum()) for m in mags) + abs(pg) + abs(kl) + 1e-30
    # |pg| terms of tokens beyond a border have no gradient: their magnitude is at most that of the bound 1 + range times |A|
    slack = ULP * kw['abs_pg']
    assert abs(float(r.policy) - pg) <= slack, (where, float(r.policy), pg)
    assert abs(float(r.kl) - kl) <= ULP * (abs(kl) + kw['abs_kl']), (where, float(r.kl), kl)
    assert abs(float(r.loss) - loss) <= slack + ULP * (abs(loss) + kw['abs_kl']) + ULP * total, (where, float(r.loss), loss)
    assert float(r.clip_fraction) == np.float32(cut), where
    assert abs(float(r.ratio) - ratio) <= ULP * abs(ratio), where


def run_policy(layout, rows, length, dtype, seed=0, adv='row', has_old=True, has_ref=True, strided=False, **kw):
    from trebi_amd.losses import policy_loss
    g, shape, which, picks = build(layout, rows, length, seed)
    base = -torch.rand(*shape, generator=g) * 3
    logp, old, ref = (base + torch.randn(*shape, generator=g) * s for s in (0.0, 0.3, 0.5))
    logp, old, ref = (v.to(DT[dtype]) for v in (logp, old, ref))
    advantages = torch.randn(*(shape if adv == 'token' else (rows,)), generator=g)
    for v in (logp, old, ref):                              # what does not count may hold anything
        keep = torch.zeros(shape, dtype=torch.bool)
        for r, p in enumerate(picks):
            (keep if keep.dim() == 1 else keep[r])[torch.from_numpy(p)] = True
        bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(DT[dtype]).min])
        v[~keep] = bad[torch.arange(int((~keep).sum())) % 4].to(DT[dtype])
    cu = [v.cuda() for v in (logp, old, ref)]
    if strided == 'transposed':
        cu = [v.t().contiguous().t() for v in cu]
    elif strided == 'slice':
        cu = [torch.cat([v, v[:, :2]], 1)[:, :length] if v.numel() else v for v in cu]
    elif strided == 'shifted':                              # contiguous, but not 16-byte aligned
        cu = [torch.cat([v.reshape(-1)[:1], v.reshape(-1)])[1:].reshape(shape) for v in cu]
    elif strided == 'columns':
        cu = [torch.stack([v, v], -1)[..., 0] for v in cu]
    r = policy_loss(cu[0], advantages.cuda(), cu[1] if has_old else None, cu[2] if has_ref else None, **which, **kw)
    A = [np.full(len(p), np64(advantages)[i]) if adv == 'row' else (np64(advantages)[p] if len(shape) == 1 else np64(advantages)[i][p])
         for i, p in enumerate(picks)]
    okw = dict(kw)
    want = F.policy(rows_of(logp, picks), A, rows_of(old, picks) if has_old else None, rows_of(ref, picks) if has_ref else None,
                    clip=okw.get('clip', 0.2), clip_high=okw.get('clip_high'), dual=okw.get('dual_clip'),
                    coef=okw.get('kl_coef', 0.0), kl=okw.get('kl', 'k3'), reduction=okw.get('reduction', 'token'),
                    denominator=okw.get('denominator'))
    big = max([1.0] + [float(np.abs(a).max()) for a in A if len(a)])
    sizes = dict(abs_pg=big * 5 * max(1.0, sum(map(len, picks)) / okw['denominator'] if okw.get('denominator') else 1.0),
                 abs_kl=20 * max(1.0, sum(map(len, picks)) / okw['denominator'] if okw.get('denominator') else 1.0))
    check_policy(r, want, picks, dtype, sizes, f'{layout} {rows}x{length} {dtype} {kw}')
    return r


LAYOUTS = ['all', 'lengths', 'mask', 'lengths mask', 'packed', 'packed-mask', 'packed-tight']


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('layout', LAYOUTS)
def test_policy_loss_matches_its_definition(layout, dtype):
    for n, (rows, length) in enumerate([(1, 1), (3, 1), (1, 7), (5, 8), (7, 20), (4, 33), (2, 600), (130, 17)]):
        run_policy(layout, rows, length, dtype, seed=n, reduction='token' if n % 2 else 'sequence', kl=('k1', 'k2', 'k3')[n % 3],
                   kl_coef=0.1, dual_clip=None if n % 2 else 3.0, adv='row' if n % 3 or layout.startswith('packed') else 'token')


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('reduction', ['token', 'sequence'])
def test_policy_loss_over_several_workgroups(layout, reduction):
    run_policy(layout, 11, 1501, 'float32', seed=4, reduction=reduction, kl_coef=0.05, clip_high=0.28)
    run_policy(layout, 700, 13, 'bfloat16', seed=5, reduction=reduction, kl_coef=0.05, clip=0.1)


@pytest.mark.parametrize('strided', ['transposed', 'slice', 'shifted', 'columns'])
@pytest.mark.parametrize('dtype', list(DT))
def test_policy_loss_reads_views(strided, dtype):
    for layout in ('all', 'lengths', 'mask'):
        run_policy(layout, 9, 21, dtype, strided=strided, kl_coef=0.1, adv='token')
    if strided in ('shifted', 'columns'):
        run_policy('packed', 9, 21, dtype, strided=strided, kl_coef=0.1)


def packed_case(lens, front, tail, seed, dtype, masked=False, adv='row', **kw):
    """A packed policy loss with the given sequence lengths against its definition."""
    from trebi_amd.losses import policy_loss
    g = torch.Generator().manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum(lens)]) + front
    n = int(cu[-1]) + tail
    base = -torch.rand(n, generator=g) * 3
    logp, old, ref = ((base + torch.randn(n, generator=g) * s).to(DT[dtype]) for s in (0.0, 0.3, 0.5))
    m = np.random.default_rng(seed).random(n) < 0.7 if masked else np.ones(n, bool)
    picks = [np.arange(cu[r], cu[r + 1])[m[cu[r]:cu[r + 1]]] for r in range(len(lens))]
    A = torch.randn(*((len(lens),) if adv == 'row' else (n,)), generator=g)
    which = dict(cu_seqlens=torch.tensor(cu, dtype=torch.int64).cuda())
    if masked:
        which['mask'] = torch.from_numpy(m).cuda()
    r = policy_loss(logp.cuda(), A.cuda(), old.cuda(), ref.cuda(), per_token=adv == 'token', **which, **kw)
    Ar = [np.full(len(p), np64(A)[i]) if adv == 'row' else np64(A)[p] for i, p in enumerate(picks)]
    want = F.policy(rows_of(logp, picks), Ar, rows_of(old, picks), rows_of(ref, picks), coef=kw.get('kl_coef', 0.0),
                    kl=kw.get('kl', 'k3'), reduction=kw.get('reduction', 'token'), dual=kw.get('dual_clip'))
    check_policy(r, want, picks, dtype, dict(abs_pg=float(A.abs().max()) * 5, abs_kl=20), (len(lens), front, tail, dtype))


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('masked', [False, True])
def test_policy_loss_packed_clusters(dtype, masked):
    """Runs of tiny and empty sequences between long ones: several in one thread's tokens, more than a wave looks at together."""
    rng = np.random.default_rng(5)
    tiny = lambda k: list(rng.integers(0, 4, size=k))
    for n, lens in enumerate([tiny(40) + [3000] + tiny(30), [5000] + tiny(300) + [1] * 50 + [4000], [0] * 200 + [2500] + [0] * 200,
                              [2, 9, 1, 0, 0, 7, 3, 1, 1, 1, 2048, 1, 2, 3, 4, 5, 6, 7, 8, 700], [1] * 3 + [4096] + [1] * 3, [6000],
                              [0, 0, 0, 6001, 0], tiny(900) + [9000]]):
        for reduction in ('token', 'sequence'):
            packed_case(lens, front=n % 3, tail=n % 5, seed=n, dtype=dtype, masked=masked, adv='token' if n % 2 else 'row',
                        reduction=reduction, kl_coef=0.1, kl=('k1', 'k2', 'k3')[n % 3], dual_clip=3.0 if n % 4 == 0 else None)


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
def test_policy_loss_every_tail(dtype):
    """Token counts one by one around a thread's, a wave's and a workgroup's share, in one workgroup and in several."""
    for n in list(range(1, 20)) + [255, 257, 511, 513, 1023, 1025, 2047, 2049, 4095, 4096, 4097, 4099, 8191, 8193, 20479, 20487]:
        packed_case([n - n // 3, n // 3], 0, 0, n, dtype)
    for L in (511, 513, 4095, 4096, 4097, 4100, 10241):
        run_policy('all', 1, L, dtype, seed=L)
        run_policy('mask', 3, L, dtype, seed=L)


def test_masks_of_other_types_and_shapes():
    from trebi_amd.losses import policy_loss, preference_loss
    g = torch.Generator('cuda').manual_seed(0)
    lp, old = (-torch.rand(6, 300, device='cuda', generator=g) for _ in range(2))
    adv = torch.randn(6, device='cuda', generator=g)
    m = torch.rand(6, 300, device='cuda', generator=g) < 0.5
    for other in (m.to(torch.uint8) * 7, m.float(), m.long(), m.t().contiguous().t()):
        a, b = policy_loss(lp, adv, old, mask=m), policy_loss(lp, adv, old, mask=other)
        assert torch.equal(a.grad, b.grad) and abs(float(a.loss) - float(b.loss)) <= 2 * ULP * float(adv.abs().max()) * 3
        p, q = preference_loss(lp, old, mask=m), preference_loss(lp, old, mask=other)
        assert torch.equal(p.grad, q.grad) and torch.equal(p.chosen_reward, q.chosen_reward)
    one = m[:1].expand(6, 300)                              # a mask that all rows share
    a, b = policy_loss(lp, adv, old, mask=one, reduction='sequence'), policy_loss(lp, adv, old, mask=one.contiguous(), reduction='sequence')
    assert not a.grad[~one].any() and (a.grad - b.grad).abs().max() <= 2 * ULP * float(adv.abs().max()) / 100
    shared = lp[:1].expand(6, 300)                          # log-probabilities that all rows share: a gradient for each
    assert policy_loss(shared, adv, shared - 0.1).grad.shape == (6, 300)
    a, b = policy_loss(lp, adv[:, None].expand(6, 300), old), policy_loss(lp, adv, old)
    assert torch.equal(a.grad, b.grad)


def test_offsets_of_64_bits_do_not_wrap():
    from trebi_amd.losses import policy_loss
    lp = -torch.rand(36, device='cuda')
    adv = torch.ones(2, device='cuda')
    a = policy_loss(lp, adv, cu_seqlens=torch.tensor([0, 7, 2 ** 32 + 3], device='cuda'))
    b = policy_loss(lp, adv, cu_seqlens=torch.tensor([0, 7, 36], device='cuda'))
    assert torch.equal(a.grad, b.grad) and a.grad.all()
    a = policy_loss(lp.view(2, 18), adv, lengths=torch.tensor([5, 2 ** 32], device='cuda'))
    assert a.grad[1].all() and not a.grad[0, 5:].any()


def test_policy_loss_without_old_or_reference_and_with_a_denominator():
    run_policy('lengths', 6, 30, 'float32', has_old=False, has_ref=False)
    run_policy('packed', 6, 30, 'bfloat16', has_old=False, kl_coef=0.2)
    run_policy('all', 6, 30, 'float32', has_ref=False, denominator=1000.0)
    run_policy('mask', 6, 30, 'float32', denominator=7.0, reduction='sequence', kl_coef=0.2)


def test_policy_loss_grad_scale_and_loss_alone():
    from trebi_amd.losses import policy_loss
    g = torch.Generator().manual_seed(0)
    logp, adv = -torch.rand(6, 50, generator=g).cuda(), torch.randn(6, generator=g).cuda()
    a, b = policy_loss(logp, adv, logp + 0.1), policy_loss(logp, adv, logp + 0.1, grad_scale=1024.0)
    assert torch.equal(a.grad * 1024.0, b.grad) and torch.equal(a.loss, b.loss)
    c = policy_loss(logp, adv, logp + 0.1, want_grad=False)
    assert c.grad is None and torch.equal(a.loss, c.loss) and torch.equal(a.ratio, c.ratio)


def test_policy_loss_nothing_valid():
    from trebi_amd.losses import policy_loss
    dev = 'cuda'
    nan = torch.full((4, 9), math.nan, device=dev)
    adv = torch.ones(4, device=dev)
    for red in ('token', 'sequence'):
        for kw in (dict(mask=torch.zeros(4, 9, dtype=torch.bool, device=dev)), dict(lengths=torch.zeros(4, dtype=torch.int64, device=dev))):
            r = policy_loss(nan, adv, nan, nan, reduction=red, kl_coef=0.1, **kw)
            assert [float(v) for v in (r.loss, r.policy, r.kl, r.clip_fraction, r.ratio)] == [0.0] * 5
            assert torch.equal(r.grad, torch.zeros_like(nan))
        cu = torch.full((5,), 3, dtype=torch.int32, device=dev)
        r = policy_loss(nan.reshape(-1), adv, cu_seqlens=cu, reduction=red)
        assert float(r.loss) == 0.0 and not r.grad.any()
    for shape in ((0, 5), (3, 0), (0,)):
        r = policy_loss(torch.zeros(shape, device=dev), torch.zeros(shape[0], device=dev))
        assert float(r.loss) == 0.0 and r.grad.shape == shape
    r = policy_loss(torch.ones(7, device=dev), torch.zeros(0, device=dev), cu_seqlens=torch.zeros(1, dtype=torch.int32, device=dev))
    assert float(r.loss) == 0.0 and not r.grad.any()


def test_policy_loss_extreme_log_probabilities():
    """-inf (an impossible token) gives ratio 0; far apart log-probabilities are held at the border; NaN comes through."""
    from trebi_amd.losses import policy_loss
    inf = math.inf
    lp = torch.tensor([[-inf, -200.0, -1.0, 0.0]], device='cuda')
    old = torch.tensor([[-1.0, -1.0, -200.0, 0.0]], device='cuda')
    r = policy_loss(lp, torch.tensor([1.0], device='cuda'), old)
    assert r.grad.tolist() == [[0.0, 0.0, 0.0, -0.25]] and abs(float(r.loss) + (0 + 0 + 1.2 + 1) / 4) < 1e-6
    r = policy_loss(lp, torch.tensor([-1.0], device='cuda'), old, dual_clip=3.0)
    assert r.grad.tolist() == [[0.0, 0.0, 0.0, 0.25]] and abs(float(r.loss) - (0.8 + 0.8 + 3 + 1) / 4) < 1e-6
    r = policy_loss(torch.tensor([[math.nan, -1.0]], device='cuda'), torch.ones(1, device='cuda'))
    assert math.isnan(float(r.loss)) and torch.isnan(r.grad).tolist() == [[True, False]]


def test_policy_loss_at_the_borders():
    """A token exactly at the border keeps its gradient, one representable step beyond loses it -- in every type."""
    from trebi_amd.losses import policy_loss
    for dtype in DT.values():
        x = torch.tensor([0.0], dtype=torch.float64)
        hi = math.log1p(0.2)
        v = torch.tensor([hi]).to(dtype)
        below = v if float(v) <= hi else torch.nextafter(v.float(), torch.tensor([-9.0])).to(dtype) if dtype == torch.float32 else (v.view(torch.int16) - 1).view(dtype)
        above = torch.nextafter(below, torch.tensor([9.0])) if dtype == torch.float32 else (below.view(torch.int16) + 1).view(dtype)
        assert float(below) <= hi < float(above)
        lp = torch.cat([below, above])[None].cuda()
        r = policy_loss(lp, torch.ones(1, device='cuda'), torch.zeros_like(lp), clip=float(np.float32(0.2)))
        # 0.2 reaches the kernel as float32: its log1p differs from log1p(0.2) by 1.5e-9, less than a step of these types
        assert (r.grad[0, 0] != 0) and (r.grad[0, 1] == 0) and float(r.clip_fraction) == 0.5


def test_policy_gradient_against_differences():
    """Central differences of the loss, in the kernel's own values: second-order error h^2 |f'''| / 6 with h = 2^-6 and third
    derivatives up to 3 |A| w, and 2 ULP of the loss / 2 h."""
    from trebi_amd.losses import policy_loss
    g = torch.Generator().manual_seed(8)
    lp = -torch.rand(3, 5, generator=g) * 2
    old, ref = lp + 0.05 * torch.randn(3, 5, generator=g), lp + 0.2 * torch.randn(3, 5, generator=g)
    adv = torch.randn(3, generator=g)
    h = 2.0 ** -6
    kw = dict(kl_coef=0.3, kl='k3', clip=0.5, reduction='sequence', lengths=torch.tensor([5, 2, 4]).cuda())
    f = lambda v: float(policy_loss(v.cuda(), adv.cuda(), old.cuda(), ref.cuda(), **kw).loss)
    grad = policy_loss(lp.cuda(), adv.cuda(), old.cuda(), ref.cuda(), **kw).grad.cpu()
    for i in range(3):
        for j in range(5):
            up, dn = lp.clone(), lp.clone()
            up[i, j] += h
            dn[i, j] -= h
            step = float(up[i, j]) - float(dn[i, j])
            bound = h * h / 6 * 4 * (float(adv.abs().max()) * 1.6 + 0.6) + 4 * 2.0 ** -23 / step
            assert abs((f(up) - f(dn)) / step - float(grad[i, j])) <= bound, (i, j)


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('strided', [False, 'columns', 'mask'])
def test_policy_loss_rows_of_one_token(strided, dtype):
    """[N, 1] and [N], with a mask, a stride between the rows, advantages one a row or one for all: as the definition says, for both means."""
    from trebi_amd.losses import policy_loss
    for N in (1, 7, 8, 9, 4096, 4097, 70001):
        g = torch.Generator().manual_seed(N)
        logp = -torch.rand(N, 3, generator=g) * 3
        old, ref = logp + 0.3 * torch.randn(N, 3, generator=g), logp + 0.3 * torch.randn(N, 3, generator=g)
        adv, mask = torch.randn(N, generator=g), torch.rand(N, 3, generator=g) < 0.7
        pick = (lambda v: v[:, 1:2]) if strided == 'columns' else (lambda v: v[:, 1:2].contiguous())
        lp, o, r = (pick(v.to(DT[dtype]).cuda()) for v in (logp, old, ref))
        m = mask.cuda()[:, 1:2] if strided else mask.cuda()[:, 1:2].contiguous()
        for use in (None, m):
            on = np.ones(N, bool) if use is None else mask[:, 1].numpy()
            out = [policy_loss(lp, adv.cuda(), o, r, mask=use, kl_coef=0.05, reduction=red) for red in ('token', 'sequence')]
            flat = policy_loss(lp[:, 0].contiguous()[None], adv.cuda()[None], o[:, 0].contiguous()[None], r[:, 0].contiguous()[None],
                               mask=None if use is None else use[:, 0].contiguous()[None], kl_coef=0.05)
            one = policy_loss(lp[:, 0], adv.cuda(), o[:, 0], r[:, 0], mask=None if use is None else use[:, 0], kl_coef=0.05)
            for v in out + [one]:
                assert v.grad.shape == (lp.shape if v is not one else (N,))
                assert torch.allclose(v.grad.reshape(-1).double(), flat.grad[0].double(), rtol=2 * F.HALF[dtype] + ULP, atol=ULP / max(on.sum(), 1))
                assert abs(float(v.loss) - float(flat.loss)) <= 2 * ULP * (1 + abs(float(flat.loss)))
    a = policy_loss(lp, torch.ones(1, device='cuda').expand(N), o, r)          # one advantage for all: stride 0
    b = policy_loss(lp, torch.ones(N, device='cuda'), o, r)
    assert torch.allclose(a.grad.float(), b.grad.float(), rtol=2 * F.HALF[dtype] + ULP, atol=0)


@pytest.mark.parametrize('reduction', ['token', 'sequence'])
@pytest.mark.parametrize('layout', ['mask', 'packed-mask'])
def test_policy_loss_counts_long_masked_rows(layout, reduction):
    run_policy(layout, 2, 70003, 'float32', seed=5, reduction=reduction, kl_coef=0.05)
    run_policy(layout, 1, 20011, 'bfloat16', seed=6, reduction=reduction)


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('which', ['all', 'lengths', 'mask'])
def test_policy_loss_sums_of_equal_ratios_have_no_bias(which, dtype):
    """Every token held at its border, with advantages of both signs and magnitude 1: the sum is one of two float32 numbers (1.28
    and 0.8 as float32), taken in float64, so only the result's own rounding is left."""
    from trebi_amd.losses import policy_loss
    R, L = 64, 1000
    adv = torch.where(torch.arange(R) % 2 == 0, 1.0, -1.0)
    old = torch.full((R, L), -1.0)
    logp = old + 0.5 * adv[:, None]
    kw, n = {}, np.full(R, L)
    if which == 'lengths':
        n = np.arange(R) * 13 + 1
        kw['lengths'] = torch.from_numpy(n).cuda()
    elif which == 'mask':
        m = np.random.default_rng(0).random((R, L)) < 0.7
        n = m.sum(1)
        kw['mask'] = torch.from_numpy(m).cuda()
    r = policy_loss(logp.to(DT[dtype]).cuda(), adv.cuda(), old.to(DT[dtype]).cuda(), clip=0.2, clip_high=0.28, **kw)
    want = np.where(np.arange(R) % 2 == 0, -float(np.float32(1 + float(np.float32(0.28)))), float(np.float32(1 - float(np.float32(0.2)))))
    want = float((want * n).sum() / n.sum())
    assert float(r.clip_fraction) == 1.0
    assert abs(float(r.policy) - want) <= F.F24 * abs(want)


@pytest.mark.parametrize('reduction', ['token', 'sequence'])
@pytest.mark.parametrize('layout', ['lengths', 'packed', 'packed-mask', 'mask'])
def test_policy_loss_counts_rows_on_both_sides_of_every_choice(layout, reduction):
    """Few rows are counted where they are needed, many by a kernel of their own; the same for calls of one workgroup."""
    for rows, length in ((2047, 5), (2048, 5), (2049, 5), (5000, 3), (4096, 1), (4097, 1), (300, 31)):
        run_policy(layout, rows, length, 'float32', seed=rows, reduction=reduction, kl_coef=0.05)


# ------------------------------------------------------------------------------------------------- preference loss
def run_pairs(layout, P, length, dtype, seed=0, strided=False, has_ref=True, weights=False, **kw):
    from trebi_amd.losses import preference_loss
    g, shape, which, picks = build(layout, 2 * P, length, seed)
    logp = -torch.rand(*shape, generator=g) * 3
    ref = logp + 0.4 * torch.randn(*shape, generator=g)
    logp, ref = logp.to(DT[dtype]), ref.to(DT[dtype])
    keep = torch.zeros(shape, dtype=torch.bool)
    for r, p in enumerate(picks):
        (keep if keep.dim() == 1 else keep[r])[torch.from_numpy(p)] = True
    for v in (logp, ref):
        v[~keep] = math.nan
    cu = [logp.cuda(), ref.cuda()]
    if strided == 'transposed':
        cu = [v.t().contiguous().t() for v in cu]
    elif strided == 'slice':
        cu = [torch.cat([v, v[:, :3]], 1)[:, :length] for v in cu]
    elif strided == 'shifted':
        cu = [torch.cat([v.reshape(-1)[:1], v.reshape(-1)])[1:].reshape(shape) for v in cu]
    w = torch.rand(P, generator=g) if weights else None
    r = preference_loss(cu[0], cu[1] if has_ref else None, weights=None if w is None else w.cuda(), **which, **kw)
    rows = rows_of(logp, picks)
    refs = rows_of(ref, picks) if has_ref else None
    beta, kind, average = kw.get('beta', 0.1), kw.get('kind', 'sigmoid'), kw.get('average', False)
    loss, rc, rr, acc, mz, gr = F.preference(rows, refs, None if w is None else np64(w), beta, kind, kw.get('label_smoothing', 0.0) if kind == 'sigmoid' else 0.0,
                                            kw.get('margin', 0.0), average, kw.get('denominator'))
    # sums in float64 of exact differences; z is rounded to float32 for the exponential (|z| 2^-24 of its value)
    D = np.concatenate([rc, rr]) / beta
    size = 1.0 + beta * np.abs(D).max() + abs(kw.get('margin', 0.0))
    got, rest = unpack(r.grad, picks)
    assert rest == 0.0
    scale = 1 / (kw.get('denominator') or P)
    for i, (a, b) in enumerate(zip(got, gr)):
        top = max(abs(b), (beta * scale if kind != 'ipo' else 0.0) / (max(len(a), 1) if average else 1))
        tol = ULP * size * top + F.HALF[dtype] * abs(b) + F.TINY[dtype]
        assert len(a) == 0 or np.abs(a - b).max() <= tol, (layout, P, length, dtype, kw, i, a[0], b)
    assert np.abs(np64(r.chosen_reward) - rc).max() <= 4 * F.F24 * max(np.abs(rc).max(), 1e-30) + 1e-12
    assert np.abs(np64(r.rejected_reward) - rr).max() <= 4 * F.F24 * max(np.abs(rr).max(), 1e-30) + 1e-12
    assert float(r.accuracy) == np.float32(acc)
    assert abs(float(r.margin) - mz) <= 4 * F.F24 * max(abs(mz), 1e-6) + 1e-12
    assert abs(float(r.loss) - loss) <= ULP * (abs(loss) + size * scale * P), (float(r.loss), loss)
    return r


@pytest.mark.parametrize('dtype', list(DT))
@pytest.mark.parametrize('layout', LAYOUTS)
def test_preference_loss_matches_its_definition(layout, dtype):
    for n, (P, length) in enumerate([(1, 1), (3, 1), (1, 7), (2, 8), (4, 20), (2, 33), (2, 600), (70, 17)]):
        run_pairs(layout, P, length, dtype, seed=n, kind=('sigmoid', 'hinge', 'ipo')[n % 3], average=bool(n % 2),
                  label_smoothing=0.1, margin=0.2 if n % 4 == 0 else 0.0, weights=n % 4 == 1, beta=(0.1, 0.5)[n % 2])


@pytest.mark.parametrize('layout', LAYOUTS)
def test_preference_loss_with_rows_split_over_workgroups(layout):
    """Few pairs of rows longer than a workgroup's turn (and, packed or with lengths, rows much shorter than the longest)."""
    for dtype in ('float32', 'bfloat16'):
        run_pairs(layout, 3, 9001, dtype, seed=2, kind='ipo', average=True)
        run_pairs(layout, 1, 20000, dtype, seed=3, beta=0.05)
    run_pairs(layout, 520, 40, 'float32', seed=4)


def test_preference_loss_many_pairs_and_every_group_size():
    for P, length in ((5000, 3), (600, 200), (513, 1500), (520, 4200)):
        run_pairs('all', P, length, 'bfloat16', seed=P, average=True)


@pytest.mark.parametrize('layout', LAYOUTS)
def test_preference_loss_on_both_sides_of_every_choice(layout):
    """Threads of a pair by the rows' lengths and the pairs' number; rows split over workgroups from 8192 tokens on."""
    for n, (P, length) in enumerate([(5, 127), (5, 129), (1023, 130), (1025, 130), (4097, 130), (4095, 130), (1025, 513), (2, 8192), (2, 8193),
                                     (70, 8200), (60, 8200)]):
        run_pairs(layout, P, length, 'float16' if n % 2 else 'float32', seed=n, average=True, weights=bool(n % 3))


@pytest.mark.parametrize('strided', ['transposed', 'slice', 'shifted'])
def test_preference_loss_reads_views_of_split_rows(strided):
    for layout in ('all', 'lengths', 'mask'):
        run_pairs(layout, 2, 9000, 'bfloat16', strided=strided, average=True)


@pytest.mark.parametrize('strided', ['transposed', 'slice', 'shifted'])
def test_preference_loss_reads_views(strided):
    for layout in ('all', 'lengths', 'mask'):
        run_pairs(layout, 4, 21, 'float32', strided=strided)
        run_pairs(layout, 2, 5000, 'bfloat16', strided=strided)


def test_preference_loss_without_reference_and_with_a_denominator():
    run_pairs('lengths', 5, 40, 'float32', has_ref=False, average=True, beta=2.0, margin=0.5)
    run_pairs('all', 5, 40, 'float32', denominator=64.0)


def test_preference_loss_empty_rows_and_batches():
    from trebi_amd.losses import preference_loss
    lp = torch.full((4, 6), math.nan, device='cuda')
    lp[1], lp[3] = -1.0, -2.0
    r = preference_loss(lp, lengths=torch.tensor([0, 6, 3, 6], device='cuda').int())       # pair 0 has an empty chosen row
    assert not r.grad[0].any() and not r.grad[2].any() and r.grad[1].all() and float(r.accuracy) == 1.0
    assert float(r.chosen_reward[0]) == 0.0
    r = preference_loss(lp, mask=torch.zeros(4, 6, dtype=torch.bool, device='cuda'))
    assert float(r.loss) == 0.0 and not r.grad.any() and float(r.margin) == 0.0
    r = preference_loss(torch.zeros(0, 6, device='cuda'))
    assert float(r.loss) == 0.0 and r.chosen_reward.shape == (0,)
    r = preference_loss(torch.zeros(4, 0, device='cuda'))
    assert float(r.loss) == 0.0 and r.grad.shape == (4, 0) and not r.chosen_reward.any()
    one = preference_loss(torch.tensor([-1.0, -2.0], device='cuda'))                        # rows of one token
    assert one.grad.shape == (2,) and float(one.accuracy) == 1.0


def test_preference_loss_far_margins():
    """Saturated pairs: the loss is linear or zero and nothing overflows; an impossible rejected row is preferred over for free."""
    from trebi_amd.losses import preference_loss
    lp = torch.tensor([[-5000.0], [0.0], [0.0], [-5000.0]], device='cuda')
    r = preference_loss(lp, beta=1.0)
    assert abs(float(r.loss) - 2500.0) < 1e-3 and r.grad[:, 0].tolist() == [-0.5, 0.0, 0.5, 0.0]
    lp = torch.tensor([[-1.0], [-math.inf]], device='cuda')
    for kind, loss in (('sigmoid', 0.0), ('hinge', 0.0)):
        r = preference_loss(lp, beta=1.0, kind=kind)
        assert float(r.loss) == loss and not r.grad.any()
    r = preference_loss(-lp.flip(0).neg(), beta=1.0, kind='hinge')
    assert float(r.loss) == math.inf and r.grad[:, 0].tolist() == [-1.0, 1.0]


def test_preference_gradient_against_differences():
    from trebi_amd.losses import preference_loss
    g = torch.Generator().manual_seed(1)
    lp, ref = -torch.rand(4, 6, generator=g) * 2, -torch.rand(4, 6, generator=g) * 2
    kw = dict(beta=0.5, label_smoothing=0.1, margin=0.1, average=True)
    f = lambda v: float(preference_loss(v.cuda(), ref.cuda(), **kw).loss)
    grad = preference_loss(lp.cuda(), ref.cuda(), **kw).grad.cpu()
    h = 2.0 ** -4
    for i in range(4):
        up, dn = lp.clone(), lp.clone()
        up[i, 2] += h
        dn[i, 2] -= h
        step = float(up[i, 2]) - float(dn[i, 2])
        # third derivative of the pair's loss in a token: at most (beta / 6)^3 / 2, /6 h^2; rounding of two losses
        assert abs((f(up) - f(dn)) / step - float(grad[i, 2])) <= h * h / 6 * (0.5 / 6) ** 3 + 2 * 2.0 ** -23 / step


# ------------------------------------------------------------------------------------------------- transitions
class Model:
    def __init__(self, T, act, obs, extra=0, epsilon=False, clamp=False):
        self.tabs = F.schedule(T)
        self.action_dim, self.observation_dim, self.transition_dim = act, obs, act + obs + extra
        self.n_timesteps, self.predict_epsilon, self.clip_denoised = T, epsilon, clamp
        for k, v in self.tabs.items():
            setattr(self, k, torch.from_numpy(v).float().cuda())


def run_transition(B, H, act, obs, T, epsilon, clamp, cond=(0,), extra=0, seed=0, chain=False):
    from trebi_amd.losses import transition_log_prob, transition_log_prob_grad
    m = Model(T, act, obs, extra, epsilon, clamp)
    D = m.transition_dim
    g = torch.Generator().manual_seed(seed)
    x, pred = torch.randn(B, H, D, generator=g), torch.randn(B, H, D, generator=g)
    t = torch.randint(0, T, (B,), generator=g)
    t[0] = 0 if B > 1 else T - 1
    xp = x + 0.1 * torch.randn(B, H, D, generator=g)
    up = torch.randn(B, generator=g)
    dx, dxp = x.cuda(), xp.cuda()
    if chain:                                               # neighbouring entries of a [B, T + 1, H, D] chain
        both = torch.stack([x, xp, x], 1).cuda()
        dx, dxp = both[:, 0], both[:, 1]
    lp = transition_log_prob(m, pred.cuda(), dx, dxp, t.cuda(), cond)
    gr = transition_log_prob_grad(m, pred.cuda(), dx, dxp, t.cuda(), up.cuda(), cond)
    want, wg, mag = F.transition(m.tabs, np64(pred), np64(x), np64(xp), t.numpy(), act, obs, set(cond), epsilon, clamp)
    # everything is float64 until one rounding to float32 (and exp(-plv) of a float64 argument): 2 roundings' worth
    assert (np.abs(np64(lp) - want) <= 2 * F.F24 * mag + 1e-30).all(), np.abs(np64(lp) - want).max()
    wg = wg * np64(up)[:, None, None]
    # the residual's own float64 rounding: a few 2^-53 of order-one terms over sigma^2 (1e10 at most) -- far below a float32 step
    assert (np.abs(np64(gr) - wg) <= 2 * F.F24 * np.abs(wg) + 1e-5 * F.F24 * np.abs(wg).max()).all()


@pytest.mark.parametrize('epsilon', [False, True])
@pytest.mark.parametrize('clamp', [False, True])
def test_transition_log_prob_matches_the_normal_density(epsilon, clamp):
    run_transition(5, 32, 6, 17, 20, epsilon, clamp)
    run_transition(3, 4, 1, 3, 20, epsilon, clamp, cond=(0, 3))
    run_transition(1, 1, 1, 1, 2, epsilon, clamp)
    run_transition(4, 7, 2, 3, 1000, epsilon, clamp, cond=(), seed=3)
    run_transition(6, 128, 6, 54, 100, epsilon, clamp, cond=(0, 5, 127, 64))          # 7680 elements: a workgroup a candidate
    run_transition(9, 5, 0, 5, 20, epsilon, clamp, extra=2, cond=(2, 2))              # the same index twice


def test_transition_takes_slices_of_a_chain():
    run_transition(6, 32, 6, 17, 20, False, False, chain=True)
    run_transition(5, 9, 2, 3, 20, True, True, chain=True)


def test_transition_more_candidates_than_workgroups():
    from trebi_amd.losses import transition_log_prob, transition_log_prob_grad
    m = Model(20, 1, 3)
    g = torch.Generator('cuda').manual_seed(2)
    B = 70001
    x, xp, pred = (torch.randn(B, 4, 4, device='cuda', generator=g) for _ in range(3))
    t = torch.randint(0, 20, (B,), device='cuda', generator=g)
    up = torch.randn(B, device='cuda', generator=g)
    lp, gr = transition_log_prob(m, pred, x, xp, t), transition_log_prob_grad(m, pred, x, xp, t, up)
    for s in (slice(0, 50), slice(40000, 40050), slice(B - 50, B)):          # the same candidates in a small batch
        assert torch.equal(lp[s], transition_log_prob(m, pred[s], x[s], xp[s], t[s]))
        assert torch.equal(gr[s], transition_log_prob_grad(m, pred[s], x[s], xp[s], t[s], up[s]))


def test_transition_empty_batch_and_refusals():
    from trebi_amd.losses import transition_log_prob, transition_log_prob_grad
    m = Model(20, 1, 3)
    z = torch.zeros(0, 4, 4, device='cuda')
    assert transition_log_prob(m, z, z, z, torch.zeros(0, dtype=torch.long)).shape == (0,)
    x = torch.zeros(2, 4, 4, device='cuda')
    with pytest.raises(ValueError):
        transition_log_prob(m, x[:, :, :3], x, x, 1)
    with pytest.raises(ValueError):
        transition_log_prob(m, x, x[:1], x, 1)
    with pytest.raises(TypeError):
        transition_log_prob(m, x, x.double(), x, 1)
    with pytest.raises(RuntimeError, match='timesteps'):
        transition_log_prob(m, x, x, x, 20)
    with pytest.raises(RuntimeError, match='outside the horizon'):
        transition_log_prob(m, x, x, x, 1, cond_keys=(4,))
    with pytest.raises(ValueError):
        transition_log_prob_grad(m, x, x, x, 1, torch.zeros(3, device='cuda'))


# ------------------------------------------------------------------------------------------------- together
def test_refusals_of_the_losses():
    from trebi_amd.losses import policy_loss, preference_loss
    x, a = torch.zeros(4, 5, device='cuda'), torch.zeros(4, device='cuda')
    for kw, err in ((dict(logp_old=x[:3]), ValueError), (dict(logp_old=x.half()), TypeError), (dict(mask=x[:, :4] > 0), ValueError),
                    (dict(lengths=torch.zeros(5, dtype=torch.int32)), ValueError), (dict(lengths=a), ValueError),
                    (dict(kl='k4'), ValueError), (dict(reduction='rows'), ValueError), (dict(clip=-1.0), RuntimeError),
                    (dict(dual_clip=0.5), RuntimeError), (dict(denominator=0.0), RuntimeError),
                    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32, device='cuda')), ValueError)):
        with pytest.raises(err):
            policy_loss(x, a, **kw)
    with pytest.raises(ValueError):
        policy_loss(x, a[:3])
    with pytest.raises(TypeError):
        policy_loss(x, a.double())
    with pytest.raises(TypeError):
        policy_loss(x.double(), a)
    with pytest.raises(ValueError, match='pairs'):
        preference_loss(x[:3])
    for kw, err in ((dict(kind='other'), ValueError), (dict(beta=0.0), RuntimeError), (dict(label_smoothing=0.7), RuntimeError),
                    (dict(weights=a), ValueError), (dict(logp_ref=x[:2]), ValueError)):
        with pytest.raises(err):
            preference_loss(x, **kw)


def test_bad_offsets_are_cut_to_the_tensor():
    """Lengths and offsets outside the tensor: as if cut (documented); nothing outside is read or written."""
    from trebi_amd.losses import policy_loss, preference_loss
    g = torch.Generator('cuda').manual_seed(0)
    lp, adv = -torch.rand(4, 9, device='cuda', generator=g), torch.randn(4, device='cuda', generator=g)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')
    a, b = policy_loss(lp, adv, lengths=i32(-5, 3, 100, 2 ** 31 - 1)), policy_loss(lp, adv, lengths=i32(0, 3, 9, 9))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)
    flat = lp.reshape(-1)
    a = policy_loss(flat, adv, cu_seqlens=i32(-7, 3, 20, 30, 2 ** 31 - 1))
    b = policy_loss(flat, adv, cu_seqlens=i32(0, 3, 20, 30, 36))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)
    a = preference_loss(flat, cu_seqlens=i32(-7, 3, 20, 30, 2 ** 31 - 1))
    b = preference_loss(flat, cu_seqlens=i32(0, 3, 20, 30, 36))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)


def test_losses_on_another_stream_and_two_at_once():
    from trebi_amd.losses import policy_loss, preference_loss
    g = torch.Generator('cuda').manual_seed(0)
    lp = [-torch.rand(64, 3000, device='cuda', generator=g) for _ in range(2)]
    adv = torch.randn(64, device='cuda', generator=g)
    mask = torch.rand(64, 3000, device='cuda', generator=g) < 0.7
    want = [(policy_loss(v, adv, v + 0.1, mask=mask), preference_loss(v, v - 0.1, mask=mask)) for v in lp]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lp]
    got = []
    for _ in range(4):
        for s, v in zip(streams, lp):
            with torch.cuda.stream(s):
                got.append((policy_loss(v, adv, v + 0.1, mask=mask), preference_loss(v, v - 0.1, mask=mask)))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        for a, b in zip(pair, want[i % 2]):
            assert torch.equal(a.loss, b.loss) and torch.equal(a.grad, b.grad)


def test_losses_captured_and_replayed():
    """Two graphs, replayed with new inputs and eager work between: every replay equals the eager result."""
    from trebi_amd.losses import policy_loss, preference_loss, transition_log_prob, transition_log_prob_grad
    g = torch.Generator('cuda').manual_seed(0)
    lp, old = (-torch.rand(40, 130, device='cuda', generator=g) for _ in range(2))
    adv = torch.randn(40, device='cuda', generator=g)
    lens = torch.randint(0, 131, (40,), device='cuda', generator=g).int()
    m = Model(20, 1, 3)
    x, xp, pred = (torch.randn(64, 4, 4, device='cuda', generator=g) for _ in range(3))
    t, up = torch.randint(0, 20, (64,), device='cuda', generator=g), torch.randn(64, device='cuda', generator=g)
    calls = [lambda: policy_loss(lp, adv, old, old, lengths=lens, reduction='sequence', kl_coef=0.1)[:3],
             lambda: preference_loss(lp, old, lengths=lens)[:3],
             lambda: (transition_log_prob(m, pred, x, xp, t), transition_log_prob_grad(m, pred, x, xp, t, up))]
    graphs = []
    for f in calls:
        f()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = f()
        graphs.append((gr, out))
    for k in range(4):
        for v in (lp, old):
            v.copy_(-torch.rand(v.shape, device='cuda', generator=g))
        pred.normal_(generator=g)
        want = [[v.clone() for v in f()] for f in calls]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b), k


def test_losses_are_reproducible_bit_for_bit():
    from trebi_amd.losses import policy_loss, preference_loss
    g = torch.Generator('cuda').manual_seed(0)
    lp = -torch.rand(300, 5001, device='cuda', generator=g)
    adv = torch.randn(300, device='cuda', generator=g)
    mask = torch.rand(300, 5001, device='cuda', generator=g) < 0.5
    a = [policy_loss(lp, adv, lp - 0.1, mask=mask, reduction='sequence') for _ in range(3)]
    b = [preference_loss(lp, mask=mask) for _ in range(3)]
    for r in a[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, a[0]))
    for r in b[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, b[0]))


def test_offsets_beyond_32_bits():
    """Rows 2^31 + 3 elements apart, and more than 2^32 tokens in one call (bfloat16, 8.6 GB each way)."""
    from trebi_amd.losses import policy_loss, preference_loss
    big = torch.empty(3 * (2 ** 31 + 3), dtype=torch.bfloat16, device='cuda')
    rows = big.as_strided((3, 5), (2 ** 31 + 3, 1))
    g = torch.Generator('cuda').manual_seed(0)
    small = -torch.rand(3, 5, device='cuda', generator=g).bfloat16()
    rows.copy_(small)
    adv = torch.randn(3, device='cuda', generator=g)
    a, b = policy_loss(rows, adv, rows), policy_loss(small, adv, small)
    assert torch.equal(a.grad, b.grad)
    # views and flat tensors sum in another order: each within the scalars' tolerance above, terms |A| w
    assert abs(float(a.loss) - float(b.loss)) <= 2 * ULP * float(adv.abs().mean())
    pa, pb = preference_loss(rows[::2]), preference_loss(small[::2])
    assert torch.equal(pa.loss, pb.loss) and torch.equal(pa.grad, pb.grad)
    del big, rows
    R, L = 5, 2 ** 30 - 3                                                    # 5.4e9 tokens
    lp = torch.zeros(R, L, dtype=torch.bfloat16, device='cuda')
    adv = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0], device='cuda')
    r = policy_loss(lp, adv, grad_scale=float(R) * L)
    assert abs(float(r.loss) + 0.6) < 1e-6
    for row in range(R):
        assert (r.grad[row] == -adv[row]).all()
    del r
    q = preference_loss(lp[:4], grad_scale=2.0 * 2, beta=1.0)                # two pairs, slopes -+ 1/2
    assert q.grad[0].eq(-1).all() and q.grad[1].eq(-1).all() and q.grad[2].eq(1).all() and q.grad[3].eq(1).all()
    lp[3, -1] = -1.0
    q = preference_loss(lp[:4], beta=1.0, want_grad=False)
    assert float(q.rejected_reward[1]) == -1.0
