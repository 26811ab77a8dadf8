"""GPU: how exact the fine-tuning losses are where errors do not average out: means over few tokens among many that do not count."""
import math

import pytest
import torch

from test_gpu_losses import DT, ULP

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
