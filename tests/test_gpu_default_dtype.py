"""GPU: what torch calls its default type (and device) is the caller's choice and reaches no result: the fine-tuning calls and
the trainer under them return the same float32 values, bit for bit, under any default."""
import contextlib

import pytest
import torch

import _finetune as F

pytestmark = pytest.mark.gpu
H, OBS, ACT, T = 8, 3, 2, 20
D = OBS + ACT


@contextlib.contextmanager
def default(dtype=None, device=None):
    before = torch.get_default_dtype()
    try:
        if dtype is not None:
            torch.set_default_dtype(dtype)
        if device is not None:
            torch.set_default_device(device)
        yield
    finally:
        torch.set_default_dtype(before)
        torch.set_default_device(None)


def losses_once(m):
    from trebi_amd.losses import policy_loss, preference_loss, transition_log_prob, transition_log_prob_grad
    f32 = dict(device='cuda', dtype=torch.float32, generator=torch.Generator('cuda').manual_seed(0))
    lp, old = -torch.rand(6, 300, **f32), -torch.rand(6, 300, **f32)
    adv = torch.randn(6, **f32)
    out = [*policy_loss(lp, adv, old, old, kl_coef=0.1, lengths=[0, 1, 300, 7, 9, 20]), *preference_loss(lp, old)]
    out += [*policy_loss(lp[:0], adv[:0]), *preference_loss(lp[:0])]
    x, xp, pred = (torch.randn(5, H, D, **f32) for _ in range(3))
    t, up = torch.tensor([0, 3, 19, 7, 1], device='cuda'), torch.randn(5, **f32)
    return out + [transition_log_prob(m, pred, x, xp, t), transition_log_prob_grad(m, pred, x, xp, t, up)]


def clip_once():
    from trebi_amd.clip import GradClipper, clip_grad_norm_
    f32 = dict(device='cuda', dtype=torch.float32, generator=torch.Generator('cuda').manual_seed(1))
    grads = [torch.randn(n, **f32) for n in (5, 4096, 70001)]
    c = GradClipper(grads)
    out = [c.norm(), *c.clip_into(1.0), c.clip_(1.0), *grads]
    p = torch.nn.Parameter(torch.zeros(9, device='cuda', dtype=torch.float32))
    p.grad = torch.full_like(p, 2.0)
    return out + [clip_grad_norm_([p], 1.0), p.grad]


def engine_once(make):
    eng, x, xp, t, adv = make
    eng.grads.zero_()
    old = eng.log_prob(x, xp, t)
    r, lp = eng.accumulate_policy(x, xp, t, adv, old, kl_coef=0.0)
    q, _ = eng.accumulate_preference(x[:2], xp[:2], t[:2])
    e, el = eng.accumulate_policy(x[:0], xp[:0], t[:0], adv[:0])
    assert eng.log_prob(x[:0], xp[:0], t[:0]).dtype == torch.float32
    one = eng.accumulate(x[:, 0], {0: x[:, 0, 0, ACT:].contiguous()}, t[:, 0], xp[:, 0])
    grads = eng.grads.clone()
    norm = eng.step(1, 0.0, max_grad_norm=1.0)
    return [old, *r, lp, *q, *e, el, one, grads, norm]


def same(a, b):
    assert len(a) == len(b)
    for u, v in zip(a, b):
        assert u.dtype == v.dtype == torch.float32 and torch.equal(u, v)


@pytest.mark.parametrize('dtype', ['float64', 'bfloat16', 'float16'])
def test_losses_and_clipping_under_another_default_type(dtype):
    from test_gpu_losses import Model
    m = Model(T, ACT, OBS)
    want = losses_once(m) + clip_once()
    with default(getattr(torch, dtype)):
        got = losses_once(m) + clip_once()
    same(want, got)


@pytest.mark.parametrize('dtype', ['float64', 'bfloat16', 'float16'])
def test_fine_tuning_under_another_default_type(dtype):
    from test_gpu_finetune import model
    diff, _ = model()
    g = torch.Generator('cuda').manual_seed(2)
    x, xp = (torch.randn(4, 3, H, D, device='cuda', generator=g) for _ in range(2))
    t, adv = torch.randint(0, T, (4, 3), device='cuda', generator=g), torch.randn(4, device='cuda', generator=g)
    want = engine_once((diff.train_engine(8), x, xp, t, adv))
    with default(getattr(torch, dtype)):
        got = engine_once((diff.train_engine(8), x, xp, t, adv))
    same(want, got)


def test_clipping_under_another_default_device():
    """The table is filled by host code: it lies in host memory whatever the default device."""
    want = clip_once()
    with default(device='cuda'):
        got = clip_once()
    same(want, got)


def plan_once(diff, noise, chain):
    from diffuser.models.diffusion import default_sample_fn
    obs = torch.linspace(-1, 1, OBS, dtype=torch.float32, device='cuda')[None].repeat(4, 1)
    out = diff.p_sample_loop((4, H, D), {0: obs}, sample_fn=default_sample_fn, verbose=False, noise=noise, return_chain=chain)
    return [v.clone() for v in (out.trajectories, out.values, *([out.chains] if chain else []))]


@pytest.mark.parametrize('dtype', ['float64', 'bfloat16', 'float16'])
def test_planning_under_another_default_type(dtype):
    from test_gpu_finetune import model
    noise = torch.randn(T + 1, 4, H, D, dtype=torch.float32, generator=torch.Generator().manual_seed(3)).cuda()
    diffs = [model()[0] for _ in range(2)]
    for chain in (False, True):
        want = plan_once(diffs[0], noise, chain)
        with default(getattr(torch, dtype)):
            got = plan_once(diffs[1], noise, chain)
            assert diffs[1].p_sample_loop((0, H, D), {0: torch.zeros(0, OBS, dtype=torch.float32, device='cuda')}).trajectories.dtype == torch.float32
        same(want, got)
