"""GPU: the gradient of every parameter through the fine-tuning losses, held to the training step's bar of 1e-3 of a gradient's
largest element in every configuration.  The log-probabilities and their gradients are taken in float64 from the library's own
prediction, so the difference between two forwards does not enter through the steep normal densities; the net's backward is the
oracle's.  And what a forward keeps for its backward."""
import numpy as np
import pytest
import torch

import _finetune as F
from test_gpu_finetune import ACT, D, H, OBS, T, Oracle, check_grads, model, split, transitions

pytestmark = pytest.mark.gpu


def chain(kw, seed, rows, steps):
    diff, sd = model(**kw)
    o = Oracle(sd, kw.get('predict_epsilon', False), kw.get('clip_denoised', False))
    x, t = transitions(rows, steps, seed)
    return diff, o, x, o.x_prev(x, t, seed + 1), t


def own_log_probs(eng, o, x, xp, t):
    """(log-probabilities, their gradients by the prediction) in float64 at the library's prediction."""
    xf, tf = torch.from_numpy(x.reshape(-1, H, D)).cuda(), torch.from_numpy(t.reshape(-1)).cuda()
    pred = torch.cat([eng.forward(xf[i:i + eng.max_batch], tf[i:i + eng.max_batch]) for i in range(0, len(xf), eng.max_batch)])
    o.forward(x, t)                                          # what the oracle's backward reads
    f64 = lambda v: v.reshape(-1, H, D).astype(np.float64)
    lp, g, _ = F.transition(o.tabs, pred.cpu().numpy().astype(np.float64), f64(x), f64(xp), t.reshape(-1), ACT, OBS, (0,), o.epsilon, o.clamp)
    return lp.reshape(t.shape), g


@pytest.mark.parametrize('max_batch', [64, 5])
@pytest.mark.parametrize('kw', [dict(), dict(predict_epsilon=True), dict(clip_denoised=True), dict(predict_epsilon=True, clip_denoised=True)])
def test_policy_gradient_at_the_library_s_own_prediction(kw, max_batch):
    rows, steps, coef = 4, 3, 0.05
    diff, o, x, xp, t = chain(kw, 15, rows, steps)
    eng = diff.train_engine(max_batch)
    lp, g = own_log_probs(eng, o, x, xp, t)
    rng = np.random.default_rng(7)
    old = (lp + rng.choice([-0.6, -0.06, 0.06, 0.6], size=lp.shape)).astype(np.float32)
    ref = (lp + 0.3 * rng.standard_normal(lp.shape)).astype(np.float32)
    adv = np.array([1.0, -1.5, 0.5, -0.7], np.float32)
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    eng.accumulate_policy(cu(x), cu(xp), cu(t), cu(adv), cu(old), cu(ref), kl_coef=coef, grad_scale=2.0)
    noisy = t > 0
    pick = lambda v: [v[i][noisy[i]].astype(np.float64) for i in range(rows)]
    gl = F.policy(pick(lp), [np.full(int(noisy[i].sum()), float(adv[i])) for i in range(rows)], pick(old), pick(ref), coef=coef)[5]
    glogp = np.zeros(lp.shape)
    glogp[noisy] = np.concatenate(gl)
    want = o.unet.backward((2.0 * glogp.reshape(-1)[:, None, None] * g).astype(np.float32), o.cache)
    check_grads(split(eng.grads, diff.model._shapes), want)


@pytest.mark.parametrize('kw', [dict(), dict(predict_epsilon=True)])
def test_preference_gradient_at_the_library_s_own_prediction(kw):
    P, steps = 3, 4
    diff, o, x, xp, t = chain(kw, 25, 2 * P, steps)
    eng = diff.train_engine(64)
    lp, g = own_log_probs(eng, o, x, xp, t)
    rng = np.random.default_rng(8)
    ref = (lp + 0.5 * rng.standard_normal(lp.shape)).astype(np.float32)
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    eng.accumulate_preference(cu(x), cu(xp), cu(t), cu(ref), beta=0.2, label_smoothing=0.1)
    noisy = t > 0
    pick = lambda v: [v[i][noisy[i]].astype(np.float64) for i in range(2 * P)]
    gr = F.preference(pick(lp), pick(ref), None, float(np.float32(0.2)), 'sigmoid', float(np.float32(0.1)))[5]
    glogp = np.where(noisy, np.array(gr)[:, None], 0.0).reshape(-1)
    want = o.unet.backward((glogp[:, None, None] * g).astype(np.float32), o.cache)
    check_grads(split(eng.grads, diff.model._shapes), want)


def test_backward_refused_after_its_inputs_changed():
    """The backward reads x and t again: changed in place since the forward, they would give another gradient."""
    diff, _ = model()
    eng = diff.train_engine(4)
    x, t = torch.zeros(4, H, D, device='cuda'), torch.ones(4, dtype=torch.long, device='cuda')
    for change in (lambda: x.add_(1.0), lambda: t.add_(1), lambda: x[1:].zero_()):
        eng.forward(x, t)
        change()
        with pytest.raises(RuntimeError, match='in place'):
            eng.backward(torch.ones_like(x))
    eng.forward(x, t)
    eng.backward(torch.ones_like(x))                         # and fine again
    with torch.inference_mode():                             # such tensors count no changes
        y = torch.zeros(4, H, D, device='cuda')
        eng.forward(y, t.clone())
        eng.backward(torch.ones_like(y))
