"""CPU: Trainer.policy_step / preference_step over two gloo ranks: every rank accumulates its own rows with the share
rows_local / rows_global, one sum over the ranks, the same clipped optimiser step everywhere."""
import os
import sys

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.join(os.path.dirname(HERE), 'safe-offline-rl-with-diffusion-model_amd')]


class _Engine:
    """Stands in for the library: the gradient of a batch is the mean of its rows (what a mean loss over rows gives)."""
    bucket_split = 0

    def __init__(self, model, max_batch):
        self.grads = torch.zeros(5)
        self.calls, self.steps = [], []

    def _add(self, x, grad_scale, **kw):
        self.calls.append((grad_scale, sorted(kw)))
        if len(x):
            self.grads += grad_scale * (x.sum(0) / kw['denominator'] if 'denominator' in kw else x.mean(0))
        return torch.zeros(()), None

    def accumulate_policy(self, x, grad_scale=1.0, **kw):
        return self._add(x, grad_scale, **kw)

    accumulate_preference = accumulate_policy

    def step(self, adam_step, lr, betas, eps, ema_mode, ema_decay, max_grad_norm=None):
        self.steps.append((adam_step, max_grad_norm, self.grads.clone()))
        self.grads.zero_()
        return torch.tensor(1.0)


class _Split(_Engine):
    bucket_split = 2


def _run(n, rank, world, engine, denominator, kind):
    from trebi_amd.parallel import shard_bounds
    from trebi_amd.training import Trainer
    tr = Trainer(None, engine_factory=engine, distributed=world > 1, max_grad_norm=0.5)
    lo, hi = shard_bounds(n, world, rank)
    batches = []
    for i in range(2):
        x = torch.from_numpy(np.random.default_rng(i).standard_normal((n, 5)).astype(np.float32))[lo:hi]
        batches.append(dict(x=x, **({'denominator': float(n)} if denominator else {})))
    step = tr.policy_step if kind == 'policy' else tr.preference_step
    step(batches, global_rows=[n, n])
    return tr.engine.steps[0], tr.step, float(tr.grad_norm)


def _worker(rank, world, port, q, *args):
    os.environ['MASTER_ADDR'] = '127.0.0.1'
    os.environ['MASTER_PORT'] = str(port)
    dist.init_process_group('gloo', rank=rank, world_size=world)
    (adam, clip, g), step, norm = _run(args[0], rank, world, *args[1:])
    q.put((rank, adam, clip, g.numpy(), step))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize('n,engine,denominator,kind', [(6, _Engine, False, 'policy'), (7, _Split, False, 'preference'),
                                                       (7, _Engine, True, 'policy'), (1, _Split, True, 'policy')])
def test_two_ranks_equal_one(n, engine, denominator, kind):
    (adam, clip, ref), step, norm = _run(n, 0, 1, engine, denominator, kind)
    assert (adam, clip, step, norm) == (1, 0.5, 1, 1.0)
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    port = 33500 + (os.getpid() + n * 3 + 11 * denominator) % 2000
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q, n, engine, denominator, kind)) for r in range(2)]
    for p in procs:
        p.start()
    outs = sorted([q.get(timeout=120) for _ in procs], key=lambda o: o[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for rank, a, c, g, s in outs:
        assert (a, c, s) == (1, 0.5, 1)
        assert np.abs(g - ref.numpy()).max() <= 8 * 2.0 ** -24 * max(1.0, np.abs(ref.numpy()).max())    # summation order
    np.testing.assert_array_equal(outs[0][3], outs[1][3])
