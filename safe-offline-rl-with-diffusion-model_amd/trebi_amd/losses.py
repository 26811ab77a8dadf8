"""Fine-tuning losses over log-probabilities, with their gradients, and the log-probability of a denoise transition, on the
HIP library (trebi_policy_loss, trebi_preference_loss, trebi_transition_logp).

Like the training step, these take no part in torch's autograd: a call returns the loss AND its gradient with respect to
the log-probabilities (times grad_scale), which the caller hands on -- TrainEngine.accumulate_policy / accumulate_preference
do so for the TemporalUnet, `logp.backward(result.grad)` does for a torch graph.  Nothing waits for the GPU, results do not
change from run to run, and the calls can be captured into a graph.  The reference has none of these losses.

Which tokens count (a token: one denoise step of a trajectory, one position of a sequence):
    logp [rows, len]                   all of them, or with lengths= [rows] a row's first ones, or / and mask= [rows, len]
    logp [tokens], cu_seqlens=         packed rows, row r at [cu_seqlens[r], cu_seqlens[r+1])  (and mask= [tokens])
    logp [rows]                        rows of one token
What stands at tokens that do not count is never used; their gradient is 0.  Inputs are float32, bfloat16 or float16 (one
type for all log-probabilities); advantages and weights float32.
"""
import ctypes as C
import struct
from collections import namedtuple

import torch

from . import _lib

PolicyLoss = namedtuple('PolicyLoss', 'loss grad policy kl clip_fraction ratio')
PreferenceLoss = namedtuple('PreferenceLoss', 'loss grad chosen_reward rejected_reward accuracy margin')

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KL = {'k1': 1, 'k2': 2, 'k3': 3}
_REDUCTIONS = {'token': 0, 'sequence': 1}
_KINDS = {'sigmoid': 0, 'hinge': 1, 'ipo': 2}


# The library's descriptors (include/trebi_hip.h), packed: a ctypes Structure of this many fields takes longer to fill than a
# small call runs on the GPU
_TOKENS = struct.Struct('@qqiPPPqq')
_POLICY = struct.Struct('@iPPPqqqqqqPqqPPffffiidf4x')
_PREFERENCE = struct.Struct('@iPPqqqqPPPPPfffiidf4x')
_TRANSITION = struct.Struct('@7i4iqqqPPPPP')
assert [v.size for v in (_TOKENS, _POLICY, _PREFERENCE, _TRANSITION)] == [
    C.sizeof(v) for v in (_lib.TokenDesc, _lib.PolicyLossDesc, _lib.PreferenceLossDesc, _lib.TransitionDesc)]


def _check_logp(logp):
    if not logp.is_cuda:
        raise RuntimeError('trebi_amd losses run on an MI355X only; there is no CPU path')
    if logp.dtype not in _DTYPES:
        raise TypeError(f'logp has type {logp.dtype}; float32, bfloat16 and float16 are supported')


def _like(name, v, logp):
    """Another per-token tensor of logp's shape, type and device."""
    if v.shape != logp.shape:
        raise ValueError(f'{name} has shape {tuple(v.shape)}, logp {tuple(logp.shape)}')
    if v.dtype is not logp.dtype:
        raise TypeError(f'{name} has type {v.dtype}, logp {logp.dtype}')
    if v.get_device() != logp.get_device():
        raise RuntimeError(f'{name} is on {v.device}, logp on {logp.device}')
    return v


def _ints(name, v, n, device):
    if not torch.is_tensor(v):
        v = torch.as_tensor(v)
    if v.shape != (n,) and n is not None or v.dim() != 1 or v.is_floating_point() or v.dtype == torch.bool:
        raise ValueError(f'{name} must be an integer tensor of shape [{n if n is not None else "rows + 1"}], got {v.dtype} {tuple(v.shape)}')
    if v.dtype is torch.int64:
        v = v.clamp(-1, 2 ** 31 - 1)                                # cut to the tensor later, but not wrapped around before
    return v.to(device, torch.int32).contiguous()


def _token_desc(logp, mask, lengths, cu_seqlens):
    """(descriptor, rows, what it points to) -- the last to be kept until the call was enqueued."""
    dev = logp.device
    keep = []
    if mask is not None:
        if mask.shape != logp.shape or mask.device != dev:
            raise ValueError(f'mask is {tuple(mask.shape)} on {mask.device}, logp {tuple(logp.shape)} on {dev}')
        if mask.dtype not in (torch.bool, torch.uint8):
            mask = mask != 0
    if cu_seqlens is not None:
        if lengths is not None:
            raise ValueError('lengths belong to padded rows, cu_seqlens to packed ones')
        if logp.dim() != 1:
            raise ValueError(f'packed logp is [tokens], got {tuple(logp.shape)}')
        cu = _ints('cu_seqlens', cu_seqlens, None, dev)
        if cu.numel() < 1:
            raise ValueError('cu_seqlens has rows + 1 entries')
        if mask is not None:
            mask = mask.contiguous()
        keep += [cu, mask]
        rows = cu.numel() - 1
        d = _TOKENS.pack(rows, logp.numel(), 1, 0, cu.data_ptr(), 0 if mask is None else mask.data_ptr(), 0, 1)
        return d, rows, keep
    rows, length = logp.shape
    if lengths is None and mask is None:
        return _TOKENS.pack(rows, length, 0, 0, 0, 0, 0, 1), rows, None
    at = None if lengths is None else _ints('lengths', lengths, rows, dev)
    ms = (0, 1) if mask is None else mask.stride()
    d = _TOKENS.pack(rows, length, 0, 0 if at is None else at.data_ptr(), 0, 0 if mask is None else mask.data_ptr(), *ms)
    return d, rows, (at, mask)


def policy_loss(logp, advantages, logp_old=None, logp_ref=None, *, mask=None, lengths=None, cu_seqlens=None, clip=0.2,
                clip_high=None, dual_clip=None, kl_coef=0.0, kl='k3', reduction='token', denominator=None, grad_scale=1.0,
                want_grad=True, per_token=None):
    """Clipped policy loss with a KL term:

        rho = exp(logp - logp_old)                       (logp_old None: on-policy, rho = 1)
        pg  = -min(rho A, clamp(rho, 1 - clip, 1 + clip_high) A),  with dual_clip c at most c |A| where A < 0
        kl  = 'k1': logp - ref | 'k2': (logp - ref)^2 / 2 | 'k3': exp(ref - logp) - (ref - logp) - 1    (no logp_ref: 0)
        loss = sum_i w_i (pg_i + kl_coef kl_i)

    w: 1 / valid tokens ('token'), 1 / (rows that are not empty * the row's valid tokens) ('sequence'), or 1 / denominator
    where that is given (data-parallel: the global count).  Nothing valid: loss 0.  advantages: one a row or one a token, told
    by their shape, or by per_token (packed rows may be as many as tokens; then one a row is assumed).
    Returns PolicyLoss(loss, grad [like logp] | None, policy, kl, clip_fraction, ratio); loss = policy + kl_coef * kl, and
    clip_fraction / ratio are means over the valid tokens."""
    _check_logp(logp)
    shape, dev = logp.shape, logp.device
    if logp.dim() == 1 and cu_seqlens is None:
        one = lambda v: v if v is None or v.dim() != 1 else v[:, None]
        if lengths is not None:
            raise ValueError('rows of one token take no lengths')
        logp, logp_old, logp_ref, mask = one(logp), one(logp_old), one(logp_ref), one(mask)
    if logp.dim() != (2 if cu_seqlens is None else 1):
        raise ValueError(f'logp is [rows, len], [rows] or (with cu_seqlens) [tokens], got {tuple(shape)}')
    if kl not in _KL or reduction not in _REDUCTIONS:
        raise ValueError(f"kl must be 'k1', 'k2' or 'k3' and reduction 'token' or 'sequence', got {kl!r}, {reduction!r}")
    if logp_old is not None:
        _like('logp_old', logp_old, logp)
    if logp_ref is not None:
        _like('logp_ref', logp_ref, logp)
    d, rows, keep = _token_desc(logp, mask, lengths, cu_seqlens)
    if advantages.dtype is not torch.float32 or advantages.get_device() != logp.get_device():
        raise TypeError(f'advantages must be float32 on {dev}, got {advantages.dtype} on {advantages.device}')
    packed = cu_seqlens is not None
    if packed:
        logp = logp.contiguous()
        logp_old = None if logp_old is None else logp_old.contiguous()
        logp_ref = None if logp_ref is None else logp_ref.contiguous()
        strides = [(0, 1)] * 3
        if advantages.shape == (rows,) and not per_token:
            adv_stride = (advantages.stride(0), 0)
        elif advantages.shape == logp.shape and per_token is not False:
            advantages, adv_stride = advantages.contiguous(), (0, 1)
        else:
            raise ValueError(f'advantages must be [{rows}] or {tuple(logp.shape)}, got {tuple(advantages.shape)}')
    else:
        strides = [logp.stride(), (0, 1) if logp_old is None else logp_old.stride(), (0, 1) if logp_ref is None else logp_ref.stride()]
        if advantages.shape in ((rows,), (rows, 1)) and (not per_token or logp.shape[1] == 1):
            adv_stride = (advantages.stride(0), 0)
        elif advantages.shape == logp.shape and per_token is not False:
            adv_stride = advantages.stride()                        # (column stride 0: one a row, expanded)
        else:
            raise ValueError(f'advantages must be [{rows}] or {tuple(logp.shape)}, got {tuple(advantages.shape)}')
    grad = torch.empty_like(logp, memory_format=torch.contiguous_format) if want_grad else None
    if rows == 0 or logp.numel() == 0:
        z = torch.zeros(5, dtype=torch.float32, device=dev).unbind()
        return PolicyLoss(z[0], None if grad is None else grad.zero_().reshape(shape), *z[1:])
    stats = torch.empty(5, dtype=torch.float32, device=dev)
    lib = _lib.lib()
    ws_bytes = lib.trebi_policy_loss_workspace_bytes(d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    q = _POLICY.pack(
        _DTYPES[logp.dtype], logp.data_ptr(), 0 if logp_old is None else logp_old.data_ptr(),
        0 if logp_ref is None else logp_ref.data_ptr(), *strides[0], *strides[1], *strides[2], advantages.data_ptr(),
        *adv_stride, 0 if grad is None else grad.data_ptr(), stats.data_ptr(), clip, clip if clip_high is None else clip_high,
        0.0 if dual_clip is None else dual_clip, kl_coef, _KL[kl], _REDUCTIONS[reduction] if denominator is None else 2,
        0.0 if denominator is None else denominator, grad_scale)
    rc = lib.trebi_policy_loss(_lib.ctx(dev.index or 0), d, q, None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream(dev))
    if rc:
        _lib.check(rc)
    loss, policy, klv, cut, ratio = stats.unbind()
    return PolicyLoss(loss, grad if grad is None or grad.shape == shape else grad.reshape(shape), policy, klv, cut, ratio)


def preference_loss(logp, logp_ref=None, *, mask=None, lengths=None, cu_seqlens=None, weights=None, beta=0.1, kind='sigmoid',
                    label_smoothing=0.0, margin=0.0, average=False, denominator=None, grad_scale=1.0, want_grad=True):
    """Preference loss over paired log ratios.  Of 2 P rows, row k is preferred to row k + P.

        D_r = sum over the row's valid tokens of logp - logp_ref   (no logp_ref: logp; average: divided by their number)
        h = D_k - D_{k+P},  z = beta h - margin
        'sigmoid': -(1 - e) log sigmoid(z) - e log sigmoid(-z), e = label_smoothing (which the other kinds do not have: no effect there)
        'hinge':   max(0, 1 - z)
        'ipo':     (z / beta - 1 / (2 beta))^2
        loss = sum_k weights[k] l_k / P     (denominator instead of P where given; data-parallel: the global number of pairs)

    A pair with an empty row gives neither loss nor gradient.  Returns PreferenceLoss(loss, grad [like logp] | None,
    chosen_reward [P], rejected_reward [P] (beta D), accuracy (share of the pairs that count with h > 0), margin (their
    mean z))."""
    _check_logp(logp)
    shape, dev = logp.shape, logp.device
    if logp.dim() == 1 and cu_seqlens is None:
        one = lambda v: v if v is None or v.dim() != 1 else v[:, None]
        if lengths is not None:
            raise ValueError('rows of one token take no lengths')
        logp, logp_ref, mask = one(logp), one(logp_ref), one(mask)
    if logp.dim() != (2 if cu_seqlens is None else 1):
        raise ValueError(f'logp is [2 P, len], [2 P] or (with cu_seqlens) [tokens], got {tuple(shape)}')
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'sigmoid', 'hinge' or 'ipo', got {kind!r}")
    if label_smoothing and kind != 'sigmoid':
        label_smoothing = 0.0                                       # the other kinds have no smoothed form
    if logp_ref is not None:
        _like('logp_ref', logp_ref, logp)
    d, rows, keep = _token_desc(logp, mask, lengths, cu_seqlens)
    if rows % 2:
        raise ValueError(f'{rows} rows: chosen and rejected rows come in pairs')
    P = rows // 2
    if weights is not None:
        if weights.shape != (P,) or weights.dtype != torch.float32 or weights.device != dev:
            raise ValueError(f'weights must be float32 [{P}] on {dev}, got {weights.dtype} {tuple(weights.shape)} on {weights.device}')
        weights = weights.contiguous()
    if cu_seqlens is not None:
        logp = logp.contiguous()
        logp_ref = None if logp_ref is None else logp_ref.contiguous()
        strides = [(0, 1)] * 2
    else:
        strides = [logp.stride(), (0, 1) if logp_ref is None else logp_ref.stride()]
    grad = torch.empty_like(logp, memory_format=torch.contiguous_format) if want_grad else None
    if P == 0:
        z = torch.zeros(3, dtype=torch.float32, device=dev).unbind()
        e = torch.empty(0, dtype=torch.float32, device=dev)
        return PreferenceLoss(z[0], None if grad is None else grad.zero_().reshape(shape), e, e.clone(), z[1], z[2])
    out = torch.empty(2 * P + 3, dtype=torch.float32, device=dev)
    lib = _lib.lib()
    ws_bytes = lib.trebi_preference_loss_workspace_bytes(d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    at = out.data_ptr()
    q = _PREFERENCE.pack(
        _DTYPES[logp.dtype], logp.data_ptr(), 0 if logp_ref is None else logp_ref.data_ptr(), *strides[0], *strides[1],
        0 if weights is None else weights.data_ptr(), 0 if grad is None else grad.data_ptr(), at, at + 4 * P, at + 8 * P, beta,
        label_smoothing, margin, _KINDS[kind], int(bool(average)), 0.0 if denominator is None else denominator, grad_scale)
    rc = lib.trebi_preference_loss(_lib.ctx(dev.index or 0), d, q, None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream(dev))
    if rc:
        _lib.check(rc)
    chosen, rejected, stats = out.split((P, P, 3))
    loss, acc, mz = stats.unbind()
    return PreferenceLoss(loss, grad if grad is None or grad.shape == shape else grad.reshape(shape), chosen, rejected, acc, mz)


# ------------------------------------------------------------------------------------------- denoise transitions
def _rows(name, v, shape, device):
    """float32 [B, H, D] whose candidates are contiguous (a slice of a chain keeps its stride), copied otherwise."""
    if v.shape != shape or v.get_device() != device:
        raise ValueError(f'{name} is {tuple(v.shape)} on {v.device}, expected {tuple(shape)} on cuda:{device}')
    if v.dtype is not torch.float32:
        raise TypeError(f'{name} must be float32, got {v.dtype}')
    s = v.stride()
    if s[2] != 1 and shape[2] > 1 or s[1] != shape[2] and shape[1] > 1:
        v = v.contiguous()
        s = v.stride()
    return v, s[0]


def _transition(model, pred, x, x_prev, t, cond_keys):
    shape, dev, T, f32 = pred.shape, pred.get_device(), model.n_timesteps, torch.float32
    if not pred.is_cuda:
        raise RuntimeError('trebi_amd computes transition log-probabilities on an MI355X only; there is no CPU path')
    if len(shape) != 3 or shape[2] != model.transition_dim:
        raise ValueError(f'pred must be [batch, horizon, {model.transition_dim}], got {tuple(shape)}')
    B, H, D = shape
    pred, ps = _rows('pred', pred, shape, dev)
    x, xs = _rows('x', x, shape, dev)
    x_prev, qs = _rows('x_prev', x_prev, shape, dev)
    if not torch.is_tensor(t):
        t = torch.as_tensor(t)
    if t.dim() == 0:
        t = t.expand(B)
    if t.dim() != 1 or t.numel() != B or t.is_floating_point():
        raise ValueError(f't must be [{B}] integers, got {t.dtype} {tuple(t.shape)}')
    if not t.is_cuda and B and not (0 <= int(t.min()) and int(t.max()) < T):
        raise RuntimeError(f'timesteps must lie in [0, {T})')
    if t.dtype is not torch.int64 or t.get_device() != dev:
        t = t.to(pred.device, torch.int64)
    t = t.contiguous()
    keys = tuple(cond_keys)
    if keys != (0,):
        keys = tuple(sorted(int(k) for k in keys))
        if len(keys) > 4:
            raise RuntimeError('at most 4 conditioned timesteps are supported')
    tables = [model.posterior_log_variance_clipped, model.posterior_mean_coef1, model.posterior_mean_coef2]
    if model.predict_epsilon:
        tables += [model.sqrt_recip_alphas_cumprod, model.sqrt_recipm1_alphas_cumprod]
    for tab in tables:
        if tab.get_device() != dev or tab.dtype is not f32 or tab.dim() != 1 or tab.numel() != T or not tab.is_contiguous():
            raise RuntimeError(f"the model's schedule must be contiguous float32 [{T}] tensors on cuda:{dev}, one is {tab.dtype} "
                               f'{tuple(tab.shape)} on {tab.device}')
    ptrs = [tab.data_ptr() for tab in tables]
    if len(ptrs) == 3:
        ptrs += [0, 0]
    d = _TRANSITION.pack(H, D, model.action_dim, model.observation_dim, T, 1 if model.clip_denoised else 0, len(keys),
                         *keys, *[0] * (4 - len(keys)), ps, xs, qs, *ptrs)
    return d, pred, x, x_prev, t


def transition_log_prob(model, pred, x, x_prev, t, cond_keys=(0,)):
    """log p(x_prev | x) [B] of the reverse step at timesteps t (GaussianDiffusion.p_mean_variance and the draw of the sample
    functions, diffusion.py:153-185), given the net's output `pred` = model.model(x, cond, t); `model` is the
    GaussianDiffusion.  Elements that a condition overwrites (observation part of the rows cond_keys) do not count, and a
    transition at t = 0, which adds no noise, has log-probability 0.  x and x_prev may be slices of a returned chain.  (A CUDA
    t is not checked here: the kernels cut it to the tables.)"""
    d, pred, x, x_prev, t = _transition(model, pred, x, x_prev, t, cond_keys)
    B, dev = pred.shape[0], pred.device
    logp = torch.empty(B, dtype=torch.float32, device=dev)
    if B:
        rc = _lib.lib().trebi_transition_logp(_lib.ctx(dev.index or 0), d, pred.data_ptr(), x.data_ptr(), x_prev.data_ptr(),
                                              t.data_ptr(), B, logp.data_ptr(), _lib.stream(dev))
        if rc:
            _lib.check(rc)
    return logp


def transition_log_prob_grad(model, pred, x, x_prev, t, grad, cond_keys=(0,)):
    """grad[b] * d transition_log_prob[b] / d pred, [B, H, D]; `grad`: float32 [B], d loss / d log-probability."""
    d, pred, x, x_prev, t = _transition(model, pred, x, x_prev, t, cond_keys)
    B, dev = pred.shape[0], pred.device
    if grad.dim() != 1 or grad.numel() != B or grad.dtype is not torch.float32 or grad.get_device() != pred.get_device():
        raise ValueError(f'grad must be float32 [{B}] on {dev}, got {grad.dtype} {tuple(grad.shape)} on {grad.device}')
    grad = grad.contiguous()
    out = torch.empty_like(pred, memory_format=torch.contiguous_format)
    if B:
        rc = _lib.lib().trebi_transition_logp_grad(_lib.ctx(dev.index or 0), d, pred.data_ptr(), x.data_ptr(), x_prev.data_ptr(),
                                                   t.data_ptr(), grad.data_ptr(), B, out.data_ptr(), _lib.stream(dev))
        if rc:
            _lib.check(rc)
    return out
