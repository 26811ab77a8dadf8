"""GPU: fine-tuning of the denoiser, end to end -- transition log-probabilities of the TemporalUnet's output, the policy or
preference loss on them, the gradient back through the net, clipping inside the optimiser step -- against the numpy oracle's net
(oracle/trebi_train_oracle.py) with the losses' float64 definitions (tests/_finetune.py) in between.

Bars.  A parameter's gradient within 1e-3 of that gradient's largest element, as for the training step, plus what the losses make of
the nets' own difference: the library's and the oracle's forward differ by at most DELTA of the largest output, and a difference
delta in the output moves a log-probability by at most sum |r| c1 / var * delta and a transition's gradient by c1 / var * delta per
element; both follow from the oracle's values, before anything is compared."""
import os
import sys

import numpy as np
import pytest
import torch

import _finetune as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'oracle'))

pytestmark = pytest.mark.gpu
H, OBS, ACT, T, DIM, MULTS = 8, 3, 2, 20, 32, (1, 2)
D = OBS + ACT
DELTA = 5e-6                       # the nets agree to 1e-5 and better (test_gpu_nets.py); half of it is a generous typical element


def model(seed=77, **kw):
    from diffuser.models import TemporalUnet, GaussianDiffusion
    from trebi_amd import spec, synth
    sd = synth.synth_state_dict(spec.unet_param_shapes(H, D, DIM, MULTS), seed)
    unet = TemporalUnet(H, D, 0, dim=DIM, dim_mults=MULTS)
    unet.load_state_dict({k: torch.from_numpy(v) for k, v in sd.items()}, strict=True)
    args = dict(n_timesteps=T, loss_type='l2', clip_denoised=False, predict_epsilon=False)
    args.update(kw)
    return GaussianDiffusion(unet, H, OBS, ACT, **args).cuda(), sd


def split(flat, shapes):
    out, off = {}, 0
    flat = flat.detach().cpu().numpy()
    for k, s in shapes.items():
        n = int(np.prod(s))
        out[k] = flat[off:off + n].reshape(s)
        off += n
    return out


def transitions(rows, steps, seed):
    """Recorded transitions: x, x_prev [rows, steps, H, D] near each other, timesteps from 3 up (and one 0), conditioned states."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, steps, H, D)).astype(np.float32)
    t = rng.integers(3, T, size=(rows, steps))
    t[0, -1] = 0
    return x, t


class Oracle:
    def __init__(self, sd, epsilon=False, clamp=False):
        import trebi_train_oracle as TO
        self.unet = TO.TrainableUnet(sd, H, D, DIM, MULTS)
        self.tabs = F.schedule(T)
        self.epsilon, self.clamp = epsilon, clamp

    def forward(self, x, t):
        self.pred, self.cache = self.unet.forward_train(x.reshape(-1, H, D), t.reshape(-1))
        return self.pred

    def x_prev(self, x, t, seed):
        """Drawn from the model itself, so that residuals are of the step's own size."""
        rng = np.random.default_rng(seed)
        pred, xf, tf = self.forward(x, t).astype(np.float64), x.reshape(-1, H, D), t.reshape(-1)
        at = lambda n: self.tabs[n][tf][:, None, None]
        x0 = at('sqrt_recip_alphas_cumprod') * xf - at('sqrt_recipm1_alphas_cumprod') * pred if self.epsilon else pred
        x0 = np.clip(x0, -1, 1) if self.clamp else x0
        mu = at('posterior_mean_coef1') * x0 + at('posterior_mean_coef2') * xf
        out = mu + np.exp(0.5 * at('posterior_log_variance_clipped')) * rng.standard_normal(mu.shape)
        return out.astype(np.float32).reshape(x.shape)

    def logp(self, x, xp, t):
        pred = self.forward(x, t).astype(np.float64)
        lp, g, mag = F.transition(self.tabs, pred, x.reshape(-1, H, D).astype(np.float64), xp.reshape(-1, H, D).astype(np.float64),
                                  t.reshape(-1), ACT, OBS, (0,), self.epsilon, self.clamp)
        delta = DELTA * np.abs(pred).max()
        self.dlogp = np.abs(g).sum((1, 2)) * delta                      # how far a log-probability may be off
        var = np.exp(self.tabs['posterior_log_variance_clipped'])
        c = self.tabs['posterior_mean_coef1'] * (self.tabs['sqrt_recipm1_alphas_cumprod'] if self.epsilon else 1.0)
        self.curve = (c ** 2 / var)[t.reshape(-1)] * delta              # ... and an element of its gradient by pred
        self.g = g
        return lp

    def backward(self, glogp):
        return self.unet.backward((glogp[:, None, None] * self.g).astype(np.float32), self.cache)


def check_grads(got, want, extra=0.0):
    for k, ref in want.items():
        ref = ref.reshape(got[k].shape)
        err = np.abs(got[k] - ref).max() / max(np.abs(ref).max(), 1e-12)
        assert err < 1e-3 + extra, (k, err, extra)


def slack(o, glogp, dglogp):
    """Relative: the net gradient of every transition may be off by the change of its log-probability's gradient, and by the
    curvature of the log-probability."""
    size = np.abs(glogp) * np.abs(o.g).max((1, 2))
    off = np.abs(dglogp) * np.abs(o.g).max((1, 2)) + np.abs(glogp) * o.curve
    return 4 * float(off.sum() / max(size.max(), 1e-30))


@pytest.mark.parametrize('max_batch', [64, 5])
@pytest.mark.parametrize('kw', [dict(), dict(predict_epsilon=True), dict(clip_denoised=True)])
def test_policy_gradient_of_every_parameter(kw, max_batch):
    diff, sd = model(**kw)
    eng = diff.train_engine(max_batch)
    o = Oracle(sd, kw.get('predict_epsilon', False), kw.get('clip_denoised', False))
    rows, steps = 4, 3
    x, t = transitions(rows, steps, 5)
    xp = o.x_prev(x, t, 6)
    lp = o.logp(x, xp, t).reshape(rows, steps)
    rng = np.random.default_rng(7)
    old = (lp + rng.choice([-0.6, -0.06, 0.06, 0.6], size=lp.shape)).astype(np.float32)       # well inside or well beyond a border
    adv = np.array([1.0, -1.5, 0.5, -0.7], np.float32)
    coef = 0.05
    ref = (lp + 0.3 * rng.standard_normal(lp.shape)).astype(np.float32)
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    r, got_lp = eng.accumulate_policy(cu(x), cu(xp), cu(t), cu(adv), cu(old), cu(ref), kl_coef=coef, grad_scale=2.0)
    noisy = t > 0
    assert np.abs(got_lp.cpu().numpy().reshape(-1) - lp.reshape(-1)).max() <= 2 * o.dlogp.max() + 1e-5 * np.abs(lp).max()
    pick = lambda v: [v[i][noisy[i]].astype(np.float64) for i in range(rows)]
    loss, _, _, _, _, g, _ = F.policy(pick(lp), [np.full(int(noisy[i].sum()), float(adv[i])) for i in range(rows)], pick(old), pick(ref), coef=coef)
    glogp = np.zeros(lp.shape)
    glogp[noisy] = np.concatenate(g)
    # |d glogp / d logp| <= w (|A| rho + coef e^delta), rho <= e^0.6, delta <= 1.5
    dg = (1.5 * 1.9 + coef * 4.5) / noisy.sum() * o.dlogp
    assert abs(float(r.loss) - loss) <= 1e-4 + float(np.abs(dg).sum())
    want = o.backward(2.0 * glogp.reshape(-1))
    check_grads(split(eng.grads, diff.model._shapes), want, slack(o, glogp.reshape(-1), dg))


def test_preference_gradient_of_every_parameter():
    diff, sd = model()
    eng = diff.train_engine(64)
    o = Oracle(sd)
    P, steps = 3, 4
    x, t = transitions(2 * P, steps, 8)
    xp = o.x_prev(x, t, 9)
    lp = o.logp(x, xp, t).reshape(2 * P, steps)
    rng = np.random.default_rng(10)
    ref = (lp + 0.5 * rng.standard_normal(lp.shape)).astype(np.float32)
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    r, _ = eng.accumulate_preference(cu(x), cu(xp), cu(t), cu(ref), beta=0.2, label_smoothing=0.1)
    noisy = t > 0
    pick = lambda v: [v[i][noisy[i]].astype(np.float64) for i in range(2 * P)]
    loss, _, _, _, _, g = F.preference(pick(lp), pick(ref), None, 0.2, 'sigmoid', 0.1)
    glogp = np.where(noisy, np.array(g)[:, None], 0.0)
    dg = 0.2 * 0.2 / 4 / P * o.dlogp.reshape(2 * P, steps).sum(1, keepdims=True) * 2 * np.ones((1, steps))   # beta^2 / 4 of the pair's change
    assert abs(float(r.loss) - loss) <= 1e-4 + 0.2 * float(o.dlogp.sum()) / P
    want = o.backward(glogp.reshape(-1))
    check_grads(split(eng.grads, diff.model._shapes), want, slack(o, glogp.reshape(-1), dg.reshape(-1)))


def test_forward_and_backward_are_the_halves_of_the_training_step():
    diff, _ = model()
    eng = diff.train_engine(16)
    g = torch.Generator('cuda').manual_seed(0)
    B = 7
    x0, noise = (torch.randn(B, H, D, device='cuda', generator=g) for _ in range(2))
    t = torch.randint(0, T, (B,), device='cuda', generator=g)
    cond = {0: x0[:, 0, ACT:].contiguous()}
    eng.accumulate(x0, cond, t, noise)
    want = eng.grads.clone()
    eng.grads.zero_()
    at = lambda v: v[t, None, None]
    xn = at(diff.sqrt_alphas_cumprod) * x0 + at(diff.sqrt_one_minus_alphas_cumprod) * noise
    xn[:, 0, ACT:] = cond[0]
    pred = eng.forward(xn, t)
    assert torch.equal(pred, eng.forward(xn, t))
    d = 2 * (pred - x0) * diff.loss_fn.weights / x0.numel()
    d[:, 0, ACT:] = 0
    eng.backward(d)
    # the same kernels on inputs that differ by a rounding (q_sample's products): 1e-4 of a gradient's largest element
    for k, v in split(eng.grads, diff.model._shapes).items():
        w = split(want, diff.model._shapes)[k]
        assert np.abs(v - w).max() <= 1e-4 * np.abs(w).max(), k


def test_halves_refuse_misuse():
    from trebi_amd import _lib
    diff, _ = model()
    eng = diff.train_engine(4)
    x, t = torch.zeros(4, H, D, device='cuda'), torch.ones(4, dtype=torch.long, device='cuda')
    with pytest.raises(RuntimeError, match='follows'):
        eng.backward(x)
    eng.forward(x, t)
    with pytest.raises(RuntimeError, match='shape'):
        eng.backward(x[:2])
    eng.backward(x)
    with pytest.raises(RuntimeError, match='follows'):
        eng.backward(x)
    eng.forward(x, t)
    eng.accumulate(x, {0: x[:, 0, ACT:]}, t, x)              # overwrites what the forward kept
    with pytest.raises(RuntimeError, match='trebi_trainer_forward'):
        eng.backward(x)
    with pytest.raises(RuntimeError, match='outside'):
        eng.forward(torch.zeros(5, H, D, device='cuda'), torch.ones(5, dtype=torch.long, device='cuda'))
    with pytest.raises(RuntimeError, match='horizon'):
        eng.forward(x[:, :4], t)
    lib = _lib.lib()
    odd = torch.zeros(4 * H * D + 1, device='cuda')[1:]
    assert lib.trebi_trainer_forward(eng.h, odd.data_ptr(), t.data_ptr(), x.data_ptr(), 4, None) == -1
    assert b'aligned' in lib.trebi_last_error()
    with pytest.raises(RuntimeError, match='timesteps'):
        eng.log_prob(x, x, torch.full((4,), T))
    with pytest.raises(RuntimeError, match='alike'):
        eng.log_prob(x, x[:3], t)


def test_backward_refused_after_the_parameters_or_the_precision_changed():
    diff, _ = model()
    eng = diff.train_engine(4)
    x, t = torch.zeros(4, H, D, device='cuda'), torch.ones(4, dtype=torch.long, device='cuda')
    for change in (eng.repack, lambda: eng.set_precision('bf16x3', 0), lambda: eng.set_precision('f32'),
                   lambda: eng.step(1, 1e-3), lambda: eng.step(2, 1e-3, max_grad_norm=1.0)):
        eng.forward(x, t)
        change()
        with pytest.raises(RuntimeError, match='trebi_trainer_forward'):
            eng.backward(x)


def test_clipped_step_equals_a_step_on_the_scaled_gradient():
    a, sd = model()
    b, _ = model()
    g = torch.Generator('cuda').manual_seed(3)
    ea, eb = a.train_engine(4), b.train_engine(4)
    for k, max_norm in enumerate((0.5, 1e6)):
        grad = torch.randn(ea.grads.numel(), device='cuda', generator=g)
        norm = float(grad.double().norm())
        ea.grads.copy_(grad)
        got = ea.step(k + 1, 1e-3, max_grad_norm=max_norm)
        assert abs(float(got) - norm) <= 2 * F.F24 * norm
        factor = torch.tensor(min(1.0, max_norm / (norm + 1e-6)), device='cuda')
        eb.grads.copy_(grad * factor)
        assert eb.step(k + 1, 1e-3) is None
        torch.cuda.synchronize()
        assert not ea.grads.any()
        # the factor may round the other way (2^-23): Adam's first and second moments then differ by as much, relatively, and the
        # parameters by 1e-3 of lr
        assert (ea.exp_avg - eb.exp_avg).abs().max() <= 4 * F.F24 * eb.exp_avg.abs().max()
        assert (ea.params - eb.params).abs().max() <= 1e-6


def test_trainer_clips_and_keeps_the_norm():
    from trebi_amd.training import Trainer
    diff, _ = model()
    g = torch.Generator('cuda').manual_seed(4)
    x = torch.randn(6, H, D, device='cuda', generator=g)
    batch = (x, {0: x[:, 0, ACT:].contiguous()}, torch.randint(0, T, (6,), device='cuda', generator=g), torch.randn(x.shape, device='cuda', generator=g))
    tr = Trainer(diff, train_batch_size=6, train_lr=1e-3, gradient_accumulate_every=1, max_grad_norm=1e-3)
    tr.engine.accumulate(*batch)
    norm = float(tr.engine.grads.double().norm())
    tr.engine.grads.zero_()
    tr.train_step([batch])
    assert abs(float(tr.grad_norm) - norm) <= 2 * F.F24 * norm
    # first step of Adam: exp_avg = 0.1 * the clipped gradient
    assert abs(float(tr.engine.exp_avg.double().norm()) - 0.1 * 1e-3) <= 1e-6 * 1e-3 + 1e-8
    plain = Trainer(model()[0], train_batch_size=6, train_lr=1e-3, gradient_accumulate_every=1)
    plain.train_step([batch])
    assert plain.grad_norm is None


def test_fine_tuning_steps_from_a_recorded_chain():
    """As they are used together: plans drawn with the chain kept, their log-probabilities, policy steps and preference steps."""
    from diffuser.models.diffusion import default_sample_fn
    from trebi_amd.training import Trainer
    diff, _ = model()
    tr = Trainer(diff, train_batch_size=32, train_lr=1e-4, gradient_accumulate_every=1, max_grad_norm=1.0)
    torch.manual_seed(0)
    R = 6
    obs = torch.randn(1, OBS, device='cuda').repeat(R, 1)
    out = diff.p_sample_loop((R, H, D), {0: obs}, sample_fn=default_sample_fn, return_chain=True, verbose=False)
    chain = out.chains
    assert chain.shape == (R, T + 1, H, D)
    x, xp, t = chain[:, :-1], chain[:, 1:], torch.arange(T - 1, -1, -1)
    old = tr.engine.log_prob(x, xp, t)
    assert old.shape == (R, T) and torch.isfinite(old).all() and not old[:, -1].any()
    # drawn from the same model: residuals are the noise, so a log-probability is that of H D - OBS normal deviates
    plv = diff.posterior_log_variance_clipped.double()[t.cuda()]
    free = H * D - OBS
    expect = -0.5 * free * (1 + np.log(2 * np.pi) + plv[:-1])
    spread = np.sqrt(free / 2)
    assert ((old[:, :-1].double() - expect).abs() <= 8 * spread).all()
    adv = torch.randn(R, device='cuda')
    before = tr.engine.params.clone()
    res = tr.policy_step([dict(x=x, x_prev=xp, t=t, advantages=adv, logp_old=old)])
    # on-policy: every ratio is 1, the loss -mean A
    assert abs(float(res[0].ratio) - 1) < 1e-3 and abs(float(res[0].loss) + float(adv.mean())) < 1e-3 * float(adv.abs().mean()) + 1e-4
    assert torch.isfinite(tr.grad_norm) and float(tr.grad_norm) > 0
    assert not torch.equal(before, tr.engine.params) and not tr.engine.grads.any() and tr.adam_steps == 1
    assert not torch.equal(tr.engine.log_prob(x, xp, t), old)
    res = tr.preference_step([dict(x=x[:4], x_prev=xp[:4], t=t, logp_ref=old[:4]), dict(x=x[2:], x_prev=xp[2:], t=t, logp_ref=old[2:])])
    assert len(res) == 2 and all(torch.isfinite(r.loss) for r in res) and tr.step == 2
    # planning goes on with the new parameters
    assert torch.isfinite(diff.p_sample_loop((R, H, D), {0: obs}, sample_fn=default_sample_fn, verbose=False).trajectories).all()


def test_empty_rows_and_steps_that_do_not_count():
    diff, _ = model()
    eng = diff.train_engine(8)
    x = torch.randn(2, 3, H, D, device='cuda')
    r, lp = eng.accumulate_policy(x, x, torch.zeros(2, 3, dtype=torch.long), torch.ones(2), lp_none(2, 3))
    assert float(r.loss) == 0.0 and not lp.any() and not eng.grads.any()
    r, lp = eng.accumulate_policy(x, x, torch.full((2, 3), 5), torch.ones(2), mask=torch.zeros(2, 3))
    assert float(r.loss) == 0.0 and not eng.grads.any()
    r, lp = eng.accumulate_policy(x[:0], x[:0], torch.zeros(0, 3, dtype=torch.long), torch.ones(0))
    assert lp.shape == (0, 3)
    r, lp = eng.accumulate_policy(x[:, 0], x[:, 0], torch.full((2,), 5), torch.ones(2))            # one step a row
    assert lp.shape == (2,) and eng.grads.any()


def lp_none(*shape):
    return torch.zeros(*shape, device='cuda')


def test_policy_accumulation_captured_and_replayed():
    diff, _ = model()
    eng = diff.train_engine(16)
    g = torch.Generator('cuda').manual_seed(0)
    x, xp = (torch.randn(3, 4, H, D, device='cuda', generator=g) for _ in range(2))
    t = torch.randint(1, T, (3, 4), device='cuda', generator=g)
    adv, old = torch.randn(3, device='cuda', generator=g), torch.zeros(3, 4, device='cuda')
    old.copy_(eng.log_prob(x, xp, t))
    call = lambda: eng.accumulate_policy(x, xp, t, adv, old, kl_coef=0.0)[0].loss
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = call()
    for k in range(4):
        x.normal_(generator=g)
        xp.copy_(x + 0.3 * torch.randn(x.shape, device='cuda', generator=g))
        adv.normal_(generator=g)
        old.copy_(eng.log_prob(x, xp, t) + 0.1)
        eng.grads.zero_()
        want_loss = call().clone()
        want = eng.grads.clone()
        eng.grads.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eng.grads, want) and torch.equal(loss, want_loss), k
