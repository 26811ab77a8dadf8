"""The denoiser's training step on the HIP library.

Reference: Trainer.train's inner step, EMA, save/load (/root/reference/diffuser/utils/training.py:19-35,37-166) and
GaussianDiffusion.loss / p_losses / q_sample (diffuser/models/diffusion.py:229-261) with WeightedL2
(diffuser/models/helpers.py:152-167,198-201).

How it maps.  The reference builds an autograd graph in `model.loss(*batch)` and walks it in `loss.backward()`; here
one library call (trebi_trainer_accumulate) does q_sample + conditioning, the TemporalUnet forward, the weighted loss
AND the whole backward, adding `grad_scale * dloss/dparams` into a flat gradient buffer.  `optimizer.step()`,
`zero_grad()` and `step_ema()` are one more call (trebi_trainer_step: torch.optim.Adam arithmetic + the EMA rule),
after which the library re-packs its kernel-layout weights from the flat parameters.

The TemporalUnet's parameters become VIEWS of one flat CUDA tensor (state_dict order, reference layouts), so
`state_dict()` / checkpoints keep working, and the data-parallel path is a single all-reduce (RCCL over xGMI) of the
3.96 M-float flat gradient per optimiser step, after all accumulation micro-batches.
"""
import ctypes as C
import os

import numpy as np
import torch
import torch.distributed as dist

from . import _lib
from .nets import TemporalUnet


def _flatten_into(module, names, flat):
    """Copy the parameters into `flat` back to back and re-point them at views of it."""
    off = 0
    for name in names:
        p = module.get_parameter(name)
        n = p.numel()
        view = flat[off:off + n].view(p.shape)
        view.copy_(p.data.to(flat.device))
        p.data = view
        off += n
    assert off == flat.numel()


def _changes(v):
    """How often a tensor was changed in place (tensors made in inference mode do not say)."""
    return None if v.is_inference() else v._version


class TrainEngine:
    """Flat parameter / gradient / Adam / EMA buffers + the library's trainer object for one GaussianDiffusion."""

    def __init__(self, diffusion, max_batch, ema_model=None, cond_keys=(0,)):
        unet = diffusion.model
        if not isinstance(unet, TemporalUnet):
            raise RuntimeError('the HIP training step covers GaussianDiffusion(TemporalUnet) (SURVEY.md 8f rank 1); '
                               f'got {type(unet).__name__}')
        kind = getattr(diffusion.loss_fn, 'kind', None)
        if kind not in ('l1', 'l2'):
            raise RuntimeError(f"loss_type {kind!r}: only the weighted 'l1' / 'l2' losses of the denoiser are built")
        dev = diffusion.betas.device
        if dev.type != 'cuda':
            raise RuntimeError('trebi_amd training runs on an MI355X only (move the model to cuda); there is no CPU path')
        self.device, self.diffusion, self.unet = dev, diffusion, unet
        self.names = list(unet._shapes.keys())
        P = sum(int(np.prod(s)) for s in unet._shapes.values())
        self.max_batch = int(max_batch)
        d = _lib.TrainDesc()
        d.horizon, d.observation_dim, d.action_dim = diffusion.horizon, diffusion.observation_dim, diffusion.action_dim
        if diffusion.transition_dim != diffusion.observation_dim + diffusion.action_dim:
            raise RuntimeError('predict_reward_done models are not built')
        d.n_timesteps, d.dim, d.n_mults = diffusion.n_timesteps, unet.dim, len(unet.dim_mults)
        for i, m in enumerate(unet.dim_mults):
            d.dim_mults[i] = m
        d.predict_epsilon = int(bool(diffusion.predict_epsilon))
        d.loss_l1 = int(kind == 'l1')
        self.cond_keys = sorted(int(k) for k in cond_keys)
        d.n_cond = len(self.cond_keys)
        for i, k in enumerate(self.cond_keys):
            d.cond_index[i] = k
        h = C.c_void_p()
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().trebi_trainer_create(_lib.ctx(dev.index or 0), C.byref(d), self.max_batch, C.byref(h)))
        self.h = h
        assert _lib.lib().trebi_trainer_param_count(h) == P
        self.params = torch.empty(P, dtype=torch.float32, device=dev)
        self.grads = torch.zeros(P, dtype=torch.float32, device=dev)
        self.exp_avg = torch.zeros(P, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(P, dtype=torch.float32, device=dev)
        _flatten_into(unet, self.names, self.params)
        self.ema = None
        if ema_model is not None:
            self.ema = torch.empty(P, dtype=torch.float32, device=dev)
            _flatten_into(ema_model.model, self.names, self.ema)
            self.ema_unet = ema_model.model
        self.loss_acc = torch.zeros(2, dtype=torch.float32, device=dev)
        tabs = [t.detach().to('cpu', torch.float32).contiguous() for t in
                (diffusion.loss_fn.weights, diffusion.sqrt_alphas_cumprod, diffusion.sqrt_one_minus_alphas_cumprod)]
        fp = lambda t: C.cast(t.data_ptr(), _lib.c_float_p)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().trebi_trainer_bind(h, _lib.ptr(self.params), _lib.ptr(self.grads), _lib.ptr(self.exp_avg),
                                                     _lib.ptr(self.exp_avg_sq), _lib.ptr(self.ema), fp(tabs[0]), fp(tabs[1]),
                                                     fp(tabs[2])))

    def _stream(self):
        return C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)

    @property
    def bucket_split(self):
        """grads[bucket_split:] (ups.*, mid_block*, final_conv.*) are final before the down path's backward runs."""
        return int(_lib.lib().trebi_trainer_bucket_split(self.h))

    def set_bucket_event(self, event):
        """`event`: a torch.cuda.Event that has been recorded once (so that its handle exists), or None.  While set,
        every accumulate() records it on its stream at the point where grads[bucket_split:] are final."""
        handle = C.c_void_p(event.cuda_event) if event is not None else C.c_void_p()
        _lib.check(_lib.lib().trebi_trainer_set_bucket_event(self.h, handle))

    def flops(self, backward=False):
        return _lib.lib().trebi_trainer_flops(self.h, 1 if backward else 0)

    def set_precision(self, mode='f32', min_batch=0):
        """Operand precision of the forward and input-gradient convolutions ('f32' | 'bf16x3', see nets.set_precision);
        the weight-gradient GEMM, the loss, Adam and the EMA stay fp32."""
        if mode not in ('f32', 'bf16x3'):
            raise ValueError("precision must be 'f32' or 'bf16x3'")
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().trebi_trainer_set_precision(self.h, 1 if mode == 'bf16x3' else 0, int(min_batch)))

    def repack(self):
        """After `params` was changed from outside (load_state_dict on the module)."""
        _lib.check(_lib.lib().trebi_trainer_repack(self.h, self._stream()))

    def accumulate(self, x, cond, t, noise, grad_scale=1.0):
        """One micro-batch: grads += grad_scale * d loss/d params.  Returns a device tensor [loss, a0_loss]."""
        B = x.shape[0]
        if B == 0:
            return torch.zeros(2, dtype=torch.float32, device=self.device)
        if sorted(int(k) for k in cond.keys()) != self.cond_keys:
            raise RuntimeError(f'conditioned timesteps {sorted(cond.keys())} differ from the engine\'s {self.cond_keys}')
        f32 = lambda v: torch.as_tensor(v, device=self.device, dtype=torch.float32).contiguous()
        x, noise = f32(x), f32(noise)
        t = torch.as_tensor(t, device=self.device).to(torch.int64).contiguous()
        cts = [f32(cond[k]) for k in self.cond_keys]
        for c in cts:
            if c.shape != (B, self.diffusion.observation_dim):
                raise RuntimeError(f'cond has shape {tuple(c.shape)}, expected {(B, self.diffusion.observation_dim)}')
        if x.shape != (B, self.diffusion.horizon, self.diffusion.transition_dim) or noise.shape != x.shape or t.shape != (B,):
            raise RuntimeError('x / noise must be [batch, horizon, transition_dim] and t [batch]')
        out = torch.zeros(2, dtype=torch.float32, device=self.device)
        _lib.check(_lib.lib().trebi_trainer_accumulate(self.h, _lib.ptr(x), _lib.ptr_array(cts), _lib.ptr(t), _lib.ptr(noise),
                                                       B, float(grad_scale), _lib.ptr(out), self._stream()))
        return out

    # ---- fine-tuning: losses over the log-probabilities of denoise transitions (trebi_amd/losses.py) ----
    def forward(self, x, t):
        """pred = unet(x, t) [B, H, D], with what backward() reads kept: B up to max_batch, x as the net is to see it.  backward() reads
        x and t again where they already are float32 / int64 and contiguous: not to be changed in place before it."""
        B = x.shape[0]
        if x.shape != (B, self.diffusion.horizon, self.diffusion.transition_dim) or t.shape != (B,):
            raise RuntimeError('x must be [batch, horizon, transition_dim] and t [batch]')
        x = x.to(self.device, torch.float32).contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        t = t.to(self.device, torch.int64).contiguous()
        pred = torch.empty_like(x)
        self._kept = None
        if B:
            _lib.check(_lib.lib().trebi_trainer_forward(self.h, _lib.ptr(x), _lib.ptr(t), _lib.ptr(pred), B, self._stream()))
            self._kept = (x, t, _changes(x), _changes(t))     # the backward reads them again
        return pred

    def backward(self, grad_pred):
        """grads += (d pred / d params)^T grad_pred, for the last forward(); once per forward()."""
        if grad_pred.shape[0] == 0:
            return
        if getattr(self, '_kept', None) is None:
            raise RuntimeError('backward() follows forward(), once')
        x, t, *changes = self._kept
        if changes != [_changes(x), _changes(t)]:
            raise RuntimeError('x or t was changed in place since forward(); backward() reads them again')
        g = grad_pred.to(self.device, torch.float32).contiguous()
        if g.shape != x.shape:
            raise RuntimeError(f'grad_pred has shape {tuple(g.shape)}, the forward\'s output {tuple(x.shape)}')
        if g.data_ptr() % 16:
            g = g.clone()
        _lib.check(_lib.lib().trebi_trainer_backward(self.h, _lib.ptr(x), _lib.ptr(t), _lib.ptr(g), x.shape[0], self._stream()))
        self._kept = None

    def _transitions(self, x, x_prev, t):
        """[rows, steps, H, D] (or [rows, H, D]: one step) and [rows, steps], [steps] or [rows] timesteps -> flat [B, H, D] x and
        x_prev, [B] t, the rows' shape."""
        x, x_prev = torch.as_tensor(x, device=self.device), torch.as_tensor(x_prev, device=self.device)
        if x.dim() not in (3, 4) or x.shape != x_prev.shape:
            raise RuntimeError(f'x and x_prev must be [rows, steps, horizon, transition_dim] alike, got {tuple(x.shape)} and {tuple(x_prev.shape)}')
        lead = tuple(x.shape[:-2])
        t = torch.as_tensor(t)
        if not t.is_cuda and t.numel() and not (0 <= int(t.min()) and int(t.max()) < self.diffusion.n_timesteps):
            raise RuntimeError(f'timesteps must lie in [0, {self.diffusion.n_timesteps})')
        t = t.to(self.device, torch.int64).expand(lead).reshape(-1)
        flat = lambda v: v.reshape(-1, *v.shape[-2:]).to(torch.float32).contiguous()
        return flat(x), flat(x_prev), t, lead

    def _parts(self, B):
        return [(lo, min(lo + self.max_batch, B)) for lo in range(0, B, self.max_batch)]

    def _fine_tune(self, x, x_prev, t, loss):
        """Log-probabilities of all transitions (micro-batches of max_batch), `loss` on them (-> an object with .grad), and its
        gradient back through the net.  The last micro-batch's forward serves its backward too; the others run again."""
        from .losses import transition_log_prob, transition_log_prob_grad
        m = self.diffusion
        x, x_prev, t, lead = self._transitions(x, x_prev, t)
        parts = self._parts(len(x))
        logp, pred = [], None
        for lo, hi in parts:
            pred = self.forward(x[lo:hi], t[lo:hi])
            logp.append(transition_log_prob(m, pred, x[lo:hi], x_prev[lo:hi], t[lo:hi], self.cond_keys))
        logp = torch.cat(logp) if logp else torch.empty(0, dtype=torch.float32, device=self.device)
        out = loss(logp.view(lead), (t > 0).view(lead))       # the last step (t = 0) adds no noise: nothing to learn from
        g = out.grad.reshape(-1)
        for k, (lo, hi) in enumerate(reversed(parts)):
            if k:
                pred = self.forward(x[lo:hi], t[lo:hi])
            self.backward(transition_log_prob_grad(m, pred, x[lo:hi], x_prev[lo:hi], t[lo:hi], g[lo:hi], self.cond_keys))
        return out, logp.view(lead)

    @torch.no_grad()
    def log_prob(self, x, x_prev, t):
        """log p(x_prev | x) of recorded transitions under the current parameters, shaped like the rows (see _transitions): what
        a policy step takes as logp_old / logp_ref.  chain[:, :-1], chain[:, 1:] and t = T-1 .. 0 are the transitions of a chain
        that p_sample_loop(return_chain=True) returned with default_sample_fn (a guide moves x between the steps)."""
        from .losses import transition_log_prob
        x, x_prev, t, lead = self._transitions(x, x_prev, t)
        out = [transition_log_prob(self.diffusion, self.forward(x[lo:hi], t[lo:hi]), x[lo:hi], x_prev[lo:hi], t[lo:hi], self.cond_keys)
               for lo, hi in self._parts(len(x))]
        self._kept = None
        return (torch.cat(out) if out else torch.empty(0, dtype=torch.float32, device=self.device)).view(lead)

    @torch.no_grad()
    def accumulate_policy(self, x, x_prev, t, advantages, logp_old=None, logp_ref=None, *, mask=None, grad_scale=1.0, **loss):
        """grads += grad_scale * d policy_loss / d params over recorded transitions (losses.policy_loss's keywords: clip,
        clip_high, dual_clip, kl_coef, kl, reduction, denominator, per_token).  x, x_prev: [rows, steps, H, D]; t: [rows, steps]
        or [steps]; advantages: one a row or one a step; logp_old / logp_ref / mask: [rows, steps].  Steps at t = 0 do not
        count.  Returns (PolicyLoss, logp [rows, steps])."""
        from .losses import policy_loss
        like = lambda v: None if v is None else torch.as_tensor(v, device=self.device, dtype=torch.float32)

        def one(logp, noisy):
            keep = noisy if mask is None else noisy & (torch.as_tensor(mask, device=self.device) != 0)
            return policy_loss(logp, like(advantages), like(logp_old), like(logp_ref), mask=keep, grad_scale=grad_scale, **loss)
        return self._fine_tune(x, x_prev, t, one)

    @torch.no_grad()
    def accumulate_preference(self, x, x_prev, t, logp_ref=None, *, mask=None, grad_scale=1.0, **loss):
        """grads += grad_scale * d preference_loss / d params (losses.preference_loss's keywords).  Rows k < rows / 2 of x, x_prev
        [rows, steps, H, D] are preferred to rows k + rows / 2; logp_ref [rows, steps]: log_prob() under the reference
        parameters.  Steps at t = 0 do not count.  Returns (PreferenceLoss, logp [rows, steps])."""
        from .losses import preference_loss
        ref = None if logp_ref is None else torch.as_tensor(logp_ref, device=self.device, dtype=torch.float32)

        def one(logp, noisy):
            keep = noisy if mask is None else noisy & (torch.as_tensor(mask, device=self.device) != 0)
            return preference_loss(logp, ref, mask=keep, grad_scale=grad_scale, **loss)
        return self._fine_tune(x, x_prev, t, one)

    def step(self, adam_step, lr, betas=(0.9, 0.999), eps=1e-8, ema_mode=0, ema_decay=0.995, max_grad_norm=None):
        """optimizer.step() and the EMA copy; with max_grad_norm the gradient is clipped to that global norm first, inside the
        same pass, and its norm before clipping returned (a device scalar)."""
        args = (self.h, int(adam_step), float(lr), float(betas[0]), float(betas[1]), float(eps), int(ema_mode), float(ema_decay))
        norm = None
        if max_grad_norm is None:
            _lib.check(_lib.lib().trebi_trainer_step(*args, self._stream()))
        else:
            norm = torch.empty((), dtype=torch.float32, device=self.device)
            _lib.check(_lib.lib().trebi_trainer_step_clipped(*args, float(max_grad_norm), _lib.ptr(norm), self._stream()))
        for net in (self.unet, getattr(self, 'ema_unet', None)):      # planning with these modules must re-pack
            if net is not None:
                net._packed_key = None
        return norm

    def __del__(self):
        try:
            torch.cuda.synchronize(self.device)
            _lib.lib().trebi_trainer_destroy(self.h)
        except Exception:
            pass


def _clone_diffusion(model):
    """copy.deepcopy(model) of training.py:61 without copying library handles: rebuild from the constructor arguments."""
    from .diffusion import GaussianDiffusion
    u = model.model
    unet = TemporalUnet(u.horizon, u.transition_dim, 0, dim=u.dim, dim_mults=u.dim_mults)
    twin = GaussianDiffusion(unet, model.horizon, model.observation_dim, model.action_dim, n_timesteps=model.n_timesteps,
                             loss_type=model.loss_type, clip_denoised=model.clip_denoised,
                             predict_epsilon=model.predict_epsilon, action_weight=model.action_weight)
    twin.load_state_dict({k: v.detach().clone() for k, v in model.state_dict().items()})
    return twin.to(model.betas.device)


def cycle(dl):                                                     # training.py:14-17
    while True:
        for data in dl:
            yield data


class Trainer:
    """diffuser.utils.training.Trainer for the denoiser (training.py:37-166): Adam, gradient accumulation, EMA,
    save / load -- rendering, wandb and cloud sync are outside the hot path and not built.

    Data-parallel: pass `group` (or have torch.distributed initialised): every rank accumulates over its own
    micro-batches, then the flat gradient is all-reduced (sum) once per optimiser step, as two slices: the tail
    bucket (up path, mid blocks, final conv: the first gradients the backward finishes) goes out on a side stream
    while the last micro-batch's down-path backward still runs, the head bucket after it.  Each micro-batch is
    scaled by B_local / B_global so that the sum equals the gradient of the mean loss over the global batch.
    max_grad_norm: clip the (reduced) gradient to that global norm in every step; `grad_norm` then holds the last one.
    policy_step / preference_step fine-tune on recorded transitions instead (no counterpart in the reference).
    `engine_factory` exists so that the distributed logic can be exercised on CPU ranks (gloo) without a GPU."""

    def __init__(self, diffusion_model, dataset=None, renderer=None, ema_decay=0.995, train_batch_size=32, train_lr=2e-5,
                 gradient_accumulate_every=2, step_start_ema=2000, update_ema_every=10, log_freq=100, sample_freq=1000,
                 save_freq=1000, label_freq=100000, save_parallel=False, results_folder='./results', n_reference=8,
                 bucket=None, group=None, distributed=None, engine_factory=None, adam_betas=(0.9, 0.999), adam_eps=1e-8,
                 max_grad_norm=None):
        self.model = diffusion_model
        self.ema_decay = ema_decay
        self.update_ema_every = update_ema_every
        self.step_start_ema = step_start_ema
        self.log_freq, self.sample_freq, self.save_freq, self.label_freq = log_freq, sample_freq, save_freq, label_freq
        self.batch_size = train_batch_size
        self.gradient_accumulate_every = gradient_accumulate_every
        self.lr, self.betas, self.eps = train_lr, adam_betas, adam_eps
        self.max_grad_norm, self.grad_norm = max_grad_norm, None
        self.dataset = dataset
        self.logdir = results_folder
        self.group = group
        self.distributed = (dist.is_available() and dist.is_initialized()) if distributed is None else distributed
        if engine_factory is None:
            self.ema_model = _clone_diffusion(diffusion_model)                       # training.py:61
            self.engine = diffusion_model.train_engine(train_batch_size, ema_model=self.ema_model)
            if self.engine.ema is None:
                raise RuntimeError('the model already has a training engine without an EMA copy')
        else:
            self.ema_model = None
            self.engine = engine_factory(diffusion_model, train_batch_size)
        self.dataloader = None
        if dataset is not None:
            self.dataloader = cycle(torch.utils.data.DataLoader(dataset, batch_size=train_batch_size, num_workers=1,
                                                                shuffle=True, pin_memory=True))
        self.step = 0
        self.adam_steps = 0
        self._bucket_event = self._side = None

    def _world(self):
        return dist.get_world_size(self.group) if self.distributed else 1

    def train_step(self, batches, global_batch_sizes=None):
        """One pass of the loop body training.py:109-122.  `batches`: gradient_accumulate_every items of
        (x, cond) or (x, cond, t, noise); t / noise are drawn like diffusion.py:260,241 when absent.
        Returns the per-micro-batch [loss, a0_loss] tensors (device, no host sync)."""
        dev = self.engine.device if hasattr(self.engine, 'device') else None
        world = self._world()
        losses = []
        g = self.engine.grads
        split = int(getattr(self.engine, 'bucket_split', 0)) if world > 1 else 0
        split = split if 0 < split < g.numel() else 0
        through_host = world > 1 and g.is_cuda and dist.get_backend(self.group) == 'gloo'
        overlap = bool(split) and g.is_cuda and not through_host
        if overlap and self._bucket_event is None:
            self._bucket_event = torch.cuda.Event()
            self._bucket_event.record(torch.cuda.current_stream(dev))      # creates the handle the library records
            self._side = torch.cuda.Stream(dev)
        tail_work = None
        for i, batch in enumerate(batches):
            x, cond = batch[0], batch[1]
            B = len(x)
            if len(batch) >= 4:
                t, noise = batch[2], batch[3]
            else:
                t = torch.randint(0, self.model.n_timesteps, (B,), device=dev).long()
                noise = torch.randn(tuple(x.shape), dtype=torch.float32, device=dev)
            Bg = global_batch_sizes[i] if global_batch_sizes is not None else B * world
            scale = (B / Bg if Bg else 0.0) / len(batches)                              # training.py:115
            last = overlap and i == len(batches) - 1
            if last:
                if B:
                    self.engine.set_bucket_event(self._bucket_event)
                else:                                      # an empty shard enqueues nothing: the stream's tail is the point
                    self._bucket_event.record(torch.cuda.current_stream(dev))
            losses.append(self.engine.accumulate(x, cond, t, noise, grad_scale=scale))
            if last:
                self.engine.set_bucket_event(None)
                self._side.wait_event(self._bucket_event)
                with torch.cuda.stream(self._side):        # the tail bucket leaves while the down path's backward runs
                    tail_work = dist.all_reduce(g[split:], op=dist.ReduceOp.SUM, group=self.group, async_op=True)
        if tail_work is not None:
            self._reduce(g[:split])
            tail_work.wait()                               # the current stream waits for the side stream's collective
        else:
            self._reduce_all()
        self._optimiser_step()
        return losses

    def _reduce(self, v):
        if v.is_cuda and dist.get_backend(self.group) == 'gloo':                        # CPU rehearsals: through the host
            vh = v.cpu()
            dist.all_reduce(vh, op=dist.ReduceOp.SUM, group=self.group)
            v.copy_(vh)
        else:
            dist.all_reduce(v, op=dist.ReduceOp.SUM, group=self.group)

    def _reduce_all(self):
        if self._world() > 1:
            g = self.engine.grads
            split = int(getattr(self.engine, 'bucket_split', 0))
            if 0 < split < g.numel():
                self._reduce(g[split:])
                self._reduce(g[:split])
            else:
                self._reduce(g)

    def _optimiser_step(self):
        self.adam_steps += 1
        ema_mode = 0
        if self.step % self.update_ema_every == 0:                                      # training.py:121-122, 94-98
            ema_mode = 1 if self.step < self.step_start_ema else 2
        clip = {} if self.max_grad_norm is None else dict(max_grad_norm=self.max_grad_norm)
        self.grad_norm = self.engine.step(self.adam_steps, self.lr, self.betas, self.eps, ema_mode, self.ema_decay, **clip)
        self.step += 1

    def _fine_tune_step(self, accumulate, batches, global_rows):
        """One optimiser step over `batches` of accumulate_policy's / accumulate_preference's arguments.  Data-parallel: every rank
        brings its own rows; each micro-batch counts rows_local / rows_global (give `denominator` for another weighting)."""
        world, out = self._world(), []
        for i, batch in enumerate(batches):
            batch = dict(batch)
            rows = len(batch['x'])
            total = global_rows[i] if global_rows is not None else rows * world
            share = 1.0 if batch.get('denominator') is not None else (rows / total if total else 0.0)
            out.append(accumulate(**batch, grad_scale=share / len(batches))[0])
        self._reduce_all()
        self._optimiser_step()
        return out

    def policy_step(self, batches, global_rows=None):
        """One clipped-policy-gradient step: `batches` are dicts of TrainEngine.accumulate_policy's arguments (x, x_prev, t,
        advantages, logp_old, ...).  Returns the per-micro-batch PolicyLoss (device, no host sync)."""
        return self._fine_tune_step(self.engine.accumulate_policy, batches, global_rows)

    def preference_step(self, batches, global_rows=None):
        """One preference step: dicts of TrainEngine.accumulate_preference's arguments (x, x_prev, t, logp_ref, ...)."""
        return self._fine_tune_step(self.engine.accumulate_preference, batches, global_rows)

    def train(self, n_train_steps):                                                     # training.py:104-139
        if self.dataloader is None:
            raise RuntimeError('Trainer.train needs a dataset; use train_step(batches) with explicit batches')
        total = []
        for _ in range(n_train_steps):
            batches = []
            for _ in range(self.gradient_accumulate_every):
                batch = next(self.dataloader)
                x, cond = batch[0], batch[1]
                batches.append((x, {int(k): v for k, v in cond.items()}))
            step = self.step
            losses = self.train_step(batches)
            total.extend(losses)
            if step % self.save_freq == 0:                  # the reference saves BEFORE `self.step += 1` (training.py:124-138)
                self.save(step // self.label_freq * self.label_freq, step=step)
            if step % self.log_freq == 0:
                l = losses[-1].tolist()
                print(f'{step}: {l[0] / self.gradient_accumulate_every:8.4f} | a0_loss: {l[1]:8.4f}', flush=True)
        print('mean loss : ', float(torch.stack(total)[:, 0].mean()))

    # ---- checkpoints in the reference's format (training.py:141-166) ----
    def save(self, epoch, step=None):
        """`step`: the value stored under 'step' (default self.step).  Data-parallel: every rank holds the same state, rank 0
        writes the file."""
        path = os.path.join(self.logdir, f'state_{epoch}.pt')
        if self.distributed and dist.get_rank(self.group) != 0:
            return path
        os.makedirs(self.logdir, exist_ok=True)
        data = {'step': self.step if step is None else step, 'model': self.model.state_dict(), 'ema': self.ema_model.state_dict()}
        torch.save({k: ({n: v.detach().cpu().clone() for n, v in d.items()} if isinstance(d, dict) else d)
                    for k, d in data.items()}, path)
        return path

    def load(self, epoch):
        path = os.path.join(self.logdir, f'state_{epoch}.pt')
        data = torch.load(path, map_location='cpu', weights_only=True)
        self.step = data['step']
        self.model.load_state_dict(data['model'])          # copies INTO the flat views
        self.ema_model.load_state_dict(data['ema'])
        self.engine.repack()
