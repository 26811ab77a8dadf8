"""GPU: the global gradient norm and clipping (trebi_amd.clip) against float64.

Tolerances: the sum is float64 and the norm one rounding (2^-24) of its root; the factor is another rounding, the product a
third: 4 * 2^-24 of a value, plus the rounding to the gradient's type (HALF) and its smallest step (TINY)."""
import math

import numpy as np
import pytest
import torch

import _finetune as F

pytestmark = pytest.mark.gpu
DT = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def make(sizes, dtypes, seed=0, scale=1.0, shift=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        v = (torch.randn(n + shift, generator=g) * scale).to(DT[dtypes[i % len(dtypes)]]).cuda()
        out.append(v[shift:])                               # shifted: aligned to the element, not to 16 bytes
    return out


def norm64(grads, kind):
    v = np.concatenate([g.detach().cpu().double().numpy().reshape(-1) for g in grads])
    if v.size == 0:
        return 0.0
    return float({2.0: np.sqrt((v * v).sum()), 1.0: np.abs(v).sum(), math.inf: np.abs(v).max()}[kind])


SIZES = [[1], [7], [0, 5, 0], [4096], [4097, 1, 255, 256, 257], [100003, 0, 31, 64, 8192, 12288], [1] * 300, [3000000, 17]]


@pytest.mark.parametrize('kind', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('dtypes', [('float32',), ('bfloat16',), ('float16',), ('float32', 'bfloat16', 'float16')])
def test_norm_and_clipping_match_float64(kind, dtypes):
    from trebi_amd.clip import GradClipper
    for k, sizes in enumerate(SIZES):
        for shift in (0, 1):
            grads = make(sizes, dtypes, seed=k, shift=shift)
            before = [g.clone() for g in grads]
            c = GradClipper(grads, kind)
            want = norm64(grads, kind)
            n = c.norm(grad_scale=0.5)
            assert abs(float(n) - 0.5 * want) <= 2 * F.F24 * want
            for max_norm in (0.25 * want, 4 * want + 1):
                factor = 0.5 * min(1.0, max_norm / (0.5 * want + 1e-6))
                flat, n2 = c.clip_into(max_norm, grad_scale=0.5)
                assert torch.equal(n, n2) and flat.shape == (sum(sizes),) and flat.dtype == torch.float32
                assert all(torch.equal(a, b) for a, b in zip(grads, before))
                got = np.split(flat.cpu().double().numpy(), np.cumsum(sizes)[:-1])
                for a, b in zip(got, before):
                    w = b.cpu().double().numpy() * factor
                    assert (np.abs(a - w) <= 4 * F.F24 * np.abs(w) + 2.0 ** -149).all()
                n3 = c.clip_(max_norm, grad_scale=0.5)
                assert torch.equal(n, n3)
                for a, b in zip(grads, before):
                    name = str(a.dtype).split('.')[1]
                    w = b.cpu().double().numpy() * factor
                    assert (np.abs(a.cpu().double().numpy() - w) <= (4 * F.F24 + F.HALF[name] * 1.001) * np.abs(w) + F.TINY[name]).all()
                for a, b in zip(grads, before):
                    a.copy_(b)


def test_within_the_norm_nothing_changes():
    from trebi_amd.clip import GradClipper
    grads = make([1000, 33], ('float32', 'bfloat16'))
    before = [g.clone() for g in grads]
    GradClipper(grads).clip_(1e9)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    GradClipper(grads).clip_(0.0)
    assert not any(g.any() for g in grads)


def test_same_as_torch():
    from trebi_amd.clip import clip_grad_norm_
    for kind in (2.0, 1.0, math.inf):
        ps = [[torch.nn.Parameter(torch.zeros(s, device='cuda')) for s in ((40, 33), (7,), (128, 64, 3))] for _ in range(2)]
        for a, b in zip(*ps):
            a.grad = torch.randn(a.shape, device='cuda')
            b.grad = a.grad.clone()
        unused = torch.nn.Parameter(torch.zeros(3, device='cuda'))
        n = clip_grad_norm_(ps[0] + [unused], 0.7, norm_type=kind)
        m = torch.nn.utils.clip_grad_norm_(ps[1], 0.7, norm_type=kind)
        assert abs(float(n) - float(m)) <= 1e-5 * float(m)                     # torch sums in float32
        for a, b in zip(*ps):
            torch.testing.assert_close(a.grad, b.grad, rtol=1e-5, atol=0)


def test_magnitudes_beyond_float32_squares():
    from trebi_amd.clip import GradClipper
    for s in (1e30, 1e-30):
        g = [torch.full((1001,), s, device='cuda')]
        n = float(GradClipper(g).norm())
        w = float(np.float32(s)) * math.sqrt(1001)
        assert abs(n - w) <= 2 * F.F24 * w


def test_infinities_and_nan():
    from trebi_amd.clip import GradClipper, clip_grad_norm_
    for kind in (2.0, 1.0, math.inf):
        for where in (0, 5000, 9999):
            a = [torch.ones(10000, device='cuda'), torch.ones(3, device='cuda')]
            a[0][where] = math.inf
            n = GradClipper(a, kind).clip_(1.0)
            assert float(n) == math.inf and float(a[1][0]) == 0.0 and math.isnan(float(a[0][where]))
            b = [torch.ones(10000, device='cuda'), torch.ones(3, device='cuda')]
            b[0][where] = math.nan
            n = GradClipper(b, kind).clip_(1.0)
            assert math.isnan(float(n)) and torch.isnan(b[1]).all()
    p = torch.nn.Parameter(torch.zeros(4, device='cuda'))
    p.grad = torch.tensor([1.0, math.inf, 0.0, 0.0], device='cuda')
    with pytest.raises(RuntimeError, match='inf'):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert float(p.grad[0]) == 1.0


def test_refusals():
    from trebi_amd.clip import GradClipper
    x = torch.zeros(8, 4, device='cuda')
    with pytest.raises(RuntimeError, match='contiguous'):
        GradClipper([x.t()])
    with pytest.raises(RuntimeError, match='overlap'):
        GradClipper([x, x])
    with pytest.raises(RuntimeError, match='overlap'):
        GradClipper([x, x[4:]])
    with pytest.raises(TypeError):
        GradClipper([x.double()])
    with pytest.raises(RuntimeError, match='is on'):
        GradClipper([x, torch.zeros(3)])
    c = GradClipper([x])
    with pytest.raises(RuntimeError, match='max_norm'):
        c.clip_(-1.0)
    with pytest.raises(RuntimeError, match='out must'):
        c.clip_into(1.0, out=torch.empty(31, device='cuda'))
    with pytest.raises(RuntimeError, match='overlaps'):
        c.clip_into(1.0, out=x.view(-1))


def test_streams_graphs_and_reproducibility():
    from trebi_amd.clip import GradClipper
    grads = make([100000, 7, 4097, 333], ('float32', 'bfloat16'), seed=1)
    c = GradClipper(grads)
    flat, n = c.clip_into(0.5)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        again = [c.clip_into(0.5) for _ in range(5)]
    mine = [c.clip_into(0.5) for _ in range(5)]             # at the same time on two streams
    torch.cuda.synchronize()
    for f, m in again + mine:
        assert torch.equal(f, flat) and torch.equal(m, n)
    work = [g.clone() for g in grads]
    cw = GradClipper(work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = cw.clip_(0.5, grad_scale=2.0)
    for k in range(4):
        fresh = make([100000, 7, 4097, 333], ('float32', 'bfloat16'), seed=10 + k)
        for a, b in zip(work, fresh):
            a.copy_(b)
        graph.replay()
        m = GradClipper(fresh).clip_(0.5, grad_scale=2.0)
        torch.cuda.synchronize()
        assert torch.equal(m, norm) and all(torch.equal(a, b) for a, b in zip(work, fresh))


def test_tensor_of_more_than_32_bit_elements():
    from trebi_amd.clip import GradClipper
    n = 2 ** 32 + 77
    a, b = torch.zeros(n, dtype=torch.bfloat16, device='cuda'), torch.ones(5, device='cuda')
    a[-1], a[0], a[2 ** 31 + 1] = 3.0, 4.0, 12.0
    c = GradClipper([a, b])
    assert float(c.norm()) == np.float32(math.sqrt(9 + 16 + 144 + 5))
    c.clip_(1.0)
    f = 1 / (math.sqrt(174) + 1e-6)
    for i, v in ((n - 1, 3.0), (0, 4.0), (2 ** 31 + 1, 12.0)):
        assert abs(float(a[i]) - v * f) <= 2.0 ** -8 * v * f + 1e-7
    assert float(a[5]) == 0.0 and abs(float(b[0]) - f) < 1e-6
