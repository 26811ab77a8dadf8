"""CPU suite: what the fine-tuning entry points refuse (argument checks come before anything touches a device), and the host
table of a gradient set."""
import ctypes as C

import numpy as np
import pytest
import torch

from trebi_amd import _lib, clip, losses

CTX = C.cast((C.c_int * 8)(), C.c_void_p)                 # only ever handed to calls that refuse their other arguments
BUF = (C.c_double * 4096)()
PTR = C.cast(BUF, C.c_void_p).value


def refused(rc, code, word):
    assert rc == code and word in _lib.lib().trebi_last_error().decode(), (rc, _lib.lib().trebi_last_error())


def tokens(**kw):
    d = _lib.TokenDesc(4, 10, 0, None, None, None, 0, 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def policy(**kw):
    q = _lib.PolicyLossDesc(0, PTR, None, None, 10, 1, 0, 0, 0, 0, PTR, 1, 0, PTR, PTR, 0.2, 0.2, 0.0, 0.0, 3, 0, 0.0, 1.0)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


def pairs(**kw):
    q = _lib.PreferenceLossDesc(0, PTR, None, 10, 1, 0, 0, None, PTR, PTR, PTR, PTR, 0.1, 0.0, 0.0, 0, 0, 0.0, 1.0)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize('change,code,word', [
    (dict(dtype=3), -1, 'type'), (dict(logp=None), -1, 'null'), (dict(advantages=None), -1, 'null'), (dict(stats=None), -1, 'null'),
    (dict(kl_kind=0), -1, 'kl_kind'), (dict(reduction=3), -1, 'reduction'), (dict(clip_low=-0.1), -1, 'clip'),
    (dict(clip_high=float('nan')), -1, 'clip'), (dict(dual_clip=0.5), -1, 'dual_clip'), (dict(dual_clip=-2.0), -1, 'dual_clip'),
    (dict(reduction=2), -1, 'denominator')])
def test_policy_loss_refuses(change, code, word):
    d, q = tokens(), policy(**change)
    refused(_lib.lib().trebi_policy_loss(CTX, C.byref(d), C.byref(q), PTR, 1 << 20, None), code, word)


@pytest.mark.parametrize('change,code,word', [
    (dict(rows=-1), -2, 'rows'), (dict(len=-1), -2, 'rows'), (dict(rows=1 << 39, len=1 << 39), -2, 'many'),
    (dict(packed=1), -1, 'cu_seqlens'), (dict(cu_seqlens=PTR), -1, 'packed'), (dict(packed=1, cu_seqlens=PTR, rows=0), -2, 'sequence'),
    (dict(packed=1, cu_seqlens=PTR, lengths=PTR), -1, 'lengths'), (dict(packed=1, cu_seqlens=PTR, len=1 << 31), -3, '32-bit'),
    (dict(packed=1, cu_seqlens=PTR, mask=PTR, mask_col_stride=2), -1, 'contiguous')])
def test_token_descriptions_refused(change, code, word):
    d = tokens(**change)
    refused(_lib.lib().trebi_policy_loss(CTX, C.byref(d), C.byref(policy()), PTR, 1 << 40, None), code, word)
    refused(_lib.lib().trebi_preference_loss(CTX, C.byref(d), C.byref(pairs()), PTR, 1 << 40, None), code, word)


def test_more_packed_sequences_than_32_bits_count_are_refused():
    lib = _lib.lib()
    for rows, code in ((0x7fffffff, -3), (1 << 39, -3)):
        d = tokens(packed=1, cu_seqlens=PTR, rows=rows)
        refused(lib.trebi_policy_loss(CTX, C.byref(d), C.byref(policy()), PTR, 1 << 50, None), code, 'fewer sequences')
        refused(lib.trebi_preference_loss(CTX, C.byref(d), C.byref(pairs()), PTR, 1 << 50, None), code, 'fewer sequences')


def test_policy_loss_refuses_masked_rows_beyond_32_bits():
    d, q = tokens(rows=1, len=1 << 31, mask=PTR), policy(reduction=1)
    refused(_lib.lib().trebi_policy_loss(CTX, C.byref(d), C.byref(q), PTR, 1 << 40, None), -3, 'masked')


def test_policy_loss_workspace_and_strides():
    lib = _lib.lib()
    assert lib.trebi_policy_loss_workspace_bytes(C.byref(tokens())) == 0      # one workgroup does it all
    d = tokens(len=100000)
    need = lib.trebi_policy_loss_workspace_bytes(C.byref(d))
    assert 0 < need < 1 << 20
    refused(lib.trebi_policy_loss(CTX, C.byref(d), C.byref(policy()), None, need, None), -1, 'null')
    refused(lib.trebi_policy_loss(CTX, C.byref(d), C.byref(policy()), PTR, need - 1, None), -4, 'workspace')
    masked = tokens(mask=PTR, rows=1000000)
    assert lib.trebi_policy_loss_workspace_bytes(C.byref(masked)) >= need + 4000000
    p = tokens(packed=1, cu_seqlens=PTR)
    refused(lib.trebi_policy_loss(CTX, C.byref(p), C.byref(policy(logp_col_stride=2)), PTR, 1 << 20, None), -3, 'contiguous')
    assert lib.trebi_policy_loss(None, C.byref(d), C.byref(policy()), PTR, 1 << 20, None) == -1


@pytest.mark.parametrize('change,code,word', [
    (dict(dtype=-1), -1, 'type'), (dict(logp=None), -1, 'null'), (dict(chosen_reward=None), -1, 'null'), (dict(kind=3), -1, 'kind'),
    (dict(beta=0.0), -1, 'beta'), (dict(beta=float('nan')), -1, 'beta'), (dict(label_smoothing=0.5), -1, 'smoothing'),
    (dict(label_smoothing=-0.1), -1, 'smoothing'), (dict(denominator=-1.0), -1, 'denominator')])
def test_preference_loss_refuses(change, code, word):
    d, q = tokens(), pairs(**change)
    refused(_lib.lib().trebi_preference_loss(CTX, C.byref(d), C.byref(q), PTR, 1 << 20, None), code, word)


def test_preference_loss_refuses_odd_rows_and_small_workspaces():
    lib = _lib.lib()
    refused(lib.trebi_preference_loss(CTX, C.byref(tokens(rows=3)), C.byref(pairs()), PTR, 1 << 20, None), -2, 'pairs')
    refused(lib.trebi_preference_loss(CTX, C.byref(tokens(rows=0)), C.byref(pairs()), PTR, 1 << 20, None), -2, 'pairs')
    d = tokens(rows=48, len=100000)
    need = lib.trebi_preference_loss_workspace_bytes(C.byref(d))
    refused(lib.trebi_preference_loss(CTX, C.byref(d), C.byref(pairs()), PTR, need - 1, None), -4, 'workspace')
    refused(lib.trebi_preference_loss(CTX, C.byref(d), C.byref(pairs()), None, need, None), -1, 'workspace')
    assert lib.trebi_preference_loss_workspace_bytes(C.byref(tokens())) == 0
    for rows, length in ((1 << 30, 1), (1 << 26, 5000)):                 # more workgroups than a launch has
        d = tokens(rows=rows, len=length)
        need = lib.trebi_preference_loss_workspace_bytes(C.byref(d))
        assert need >= rows // 2 // 16 * 32
        refused(lib.trebi_preference_loss(CTX, C.byref(d), C.byref(pairs()), PTR, need, None), -3, 'pairs')


def transition(**kw):
    d = _lib.TransitionDesc(8, 5, 2, 3, 20, 0, 1, (C.c_int * 4)(0), 40, 40, 40, PTR, PTR, PTR, None, None)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize('change,code,word', [
    (dict(horizon=0), -2, 'dimensions'), (dict(action_dim=3), -2, 'dimensions'), (dict(n_timesteps=0), -2, 'dimensions'),
    (dict(horizon=1 << 28), -2, 'dimensions'), (dict(posterior_log_variance=None), -1, 'table'), (dict(coef2=None), -1, 'table'),
    (dict(sqrt_recip_alphas_cumprod=PTR), -1, 'together'), (dict(n_cond=5), -3, '4'), (dict(cond_index=(C.c_int * 4)(8)), -2, 'horizon'),
    (dict(cond_index=(C.c_int * 4)(-1)), -2, 'horizon')])
def test_transitions_refused(change, code, word):
    lib = _lib.lib()
    d = transition(**change)
    refused(lib.trebi_transition_logp(CTX, C.byref(d), PTR, PTR, PTR, PTR, 4, PTR, None), code, word)
    refused(lib.trebi_transition_logp_grad(CTX, C.byref(d), PTR, PTR, PTR, PTR, PTR, 4, PTR, None), code, word)


def test_transitions_refuse_null_tensors_and_take_empty_batches():
    lib, d = _lib.lib(), transition()
    refused(lib.trebi_transition_logp(CTX, C.byref(d), None, PTR, PTR, PTR, 4, PTR, None), -1, 'null')
    refused(lib.trebi_transition_logp(CTX, C.byref(d), PTR, PTR, PTR, PTR, 4, None, None), -1, 'null')
    refused(lib.trebi_transition_logp_grad(CTX, C.byref(d), PTR, PTR, PTR, PTR, None, 4, PTR, None), -1, 'null')
    refused(lib.trebi_transition_logp(CTX, C.byref(d), PTR, PTR, PTR, PTR, -1, PTR, None), -2, 'batch')
    assert lib.trebi_transition_logp(CTX, C.byref(d), None, None, None, None, 0, None, None) == 0


def fill(ptrs, numels, dtypes, table=None, short=0):
    lib, n = _lib.lib(), len(numels)
    nm = (C.c_int64 * n)(*numels)
    size = lib.trebi_grad_set_bytes(n, nm)
    buf = np.zeros(size // 8 + 1, np.int64)
    s = _lib.GradSet()
    rc = lib.trebi_grad_set_fill(n, (C.c_void_p * n)(*ptrs), nm, (C.c_int * n)(*dtypes), buf.ctypes.data, size - short, C.byref(s))
    return rc, s, buf


@pytest.mark.parametrize('numels', [[0, 1, 7, 4096, 4097, 100000, 0, 33, 12289], [0], [1], [5] * 700, [20000000, 0, 3], [0] * 9,
                                    [3584, 3585, 3583, 512, 0, 4096]])
def test_gradient_set_table_covers_every_element_once(numels):
    rng = np.random.default_rng(3)
    starts, at = [], 1 << 20
    for n in numels:
        starts.append(at)
        at += 4 * n + 4 * int(rng.integers(0, 5))
    rc, s, buf = fill(starts, numels, [0] * len(numels))
    assert rc == 0 and s.n_tensors == len(numels) and s.total == sum(numels) and s.bytes == 4 * s.total
    ch = buf.view(np.uint8)[:24 * s.n_chunks].view(np.dtype([('p', '<u8'), ('out', '<i8'), ('len', '<i4'), ('dtype', '<i4')]))
    seen = [np.zeros(n, int) for n in numels]
    first = np.cumsum([0] + numels)
    for c in ch:
        i = int(np.searchsorted(first, c['out'], side='right')) - 1        # the tensor (not empty) that the chunk's output lies in
        off = int(c['out']) - int(first[i])
        assert c['len'] > 0 and c['dtype'] == 0 and int(c['p']) == starts[i] + 4 * off and off + c['len'] <= numels[i]
        seen[i][off:off + c['len']] += 1
    assert all((v == 1).all() for v in seen)


def test_gradient_sets_refused():
    rc, _, _ = fill([1024, 1024], [4, 4], [0, 0])
    refused(rc, -1, 'overlap')                                             # the same tensor twice
    rc, _, _ = fill([1024, 1036], [4, 4], [0, 0])
    refused(rc, -1, 'overlap')
    rc, _, _ = fill([1024, 1032], [4, 4], [1, 0])                          # touching ends are fine
    assert rc == 0
    rc, _, _ = fill([1026], [4], [0])
    refused(rc, -1, 'aligned')
    rc, _, _ = fill([None], [4], [0])
    refused(rc, -1, 'null')
    rc, _, _ = fill([1024], [4], [3])
    refused(rc, -1, 'type')
    rc, _, _ = fill([1024], [4], [0], short=1)
    refused(rc, -4, 'table')
    lib = _lib.lib()
    assert lib.trebi_grad_set_bytes(1, (C.c_int64 * 1)(-1)) == 0 and lib.trebi_grad_set_bytes(0, None) == 0


@pytest.mark.parametrize('kw,code,word', [(dict(norm=3), -1, 'norm_type'), (dict(scale=-1.0), -1, 'grad_scale'), (dict(scale=float('nan')), -1, 'grad_scale'),
                                          (dict(ws=8), -4, 'workspace'), (dict(max_norm=-1.0), -1, 'max_norm'), (dict(max_norm=float('nan')), -1, 'max_norm')])
def test_clipping_refused(kw, code, word):
    lib = _lib.lib()
    rc, s, _ = fill([1024], [4], [0])
    assert rc == 0
    a = dict(norm=0, scale=1.0, ws=1 << 20, max_norm=1.0)
    a.update(kw)
    refused(lib.trebi_grad_clip(CTX, C.byref(s), PTR, a['norm'], a['max_norm'], a['scale'], None, PTR, PTR, a['ws'], None), code, word)
    if 'max_norm' not in kw:
        refused(lib.trebi_grad_norm(CTX, C.byref(s), PTR, a['norm'], a['scale'], PTR, PTR, a['ws'], None), code, word)


def test_python_refuses_cpu_tensors_and_unknown_names():
    z = torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match='MI355X'):
        losses.policy_loss(z, torch.zeros(4))
    with pytest.raises(RuntimeError, match='MI355X'):
        losses.preference_loss(z)
    with pytest.raises(RuntimeError, match='MI355X'):
        clip.GradClipper([z])
    with pytest.raises(ValueError, match='at least one'):
        clip.GradClipper([])
    with pytest.raises(ValueError, match='norm_type'):
        clip.GradClipper([z], norm_type=3)
    assert float(clip.clip_grad_norm_([torch.nn.Parameter(z)], 1.0)) == 0.0        # no gradients at all
