"""Global gradient norm over many tensors, and clipping, on the HIP library (trebi_grad_*).

    clipper = GradClipper(grads)                    # once: the tensors stay where they are from step to step
    norm = clipper.clip_(1.0)                       # per step: in place, two launches whatever the number of tensors
    flat, norm = clipper.clip_into(1.0, grad_scale=1 / loss_scale)   # float32 copies, back to back, gradients untouched

With s = grad_scale:  n = s * ||all gradients||,  every gradient becomes s * min(1, max_norm / (n + 1e-6)) * g
(torch.nn.utils.clip_grad_norm_'s arithmetic; the sum is taken in float64).  The norm comes back as a device tensor: a
GradClipper's calls do not wait for the GPU.  Making one does (its table is copied to the device), and so does the function
clip_grad_norm_, which makes one in every call.  training.Trainer(max_grad_norm=...) clips its flat gradient inside the
optimiser step instead.
The reference trains without clipping.
"""
import ctypes as C
import math

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _norm_kind(norm_type):
    kind = {2.0: 0, 1.0: 1, math.inf: 2}.get(float(norm_type))
    if kind is None:
        raise ValueError(f'norm_type must be 2, 1 or inf, got {norm_type}')
    return kind


class GradClipper:
    """Bound to a list of CUDA gradients (float32, bfloat16 and float16 may be mixed; contiguous; none twice): holds them and
    the device table of their places.  Make a new one when a gradient is allocated anew (zero_grad(set_to_none=True), torch's
    default, leaves .grad to be: this one would go on with the old tensors), and keep it as long as graphs that captured its calls.  Making one copies the table to the device, so it cannot be captured; the calls can."""

    def __init__(self, tensors, norm_type=2.0):
        self.tensors = list(tensors)
        self.norm_type = _norm_kind(norm_type)
        if not self.tensors:
            raise ValueError('GradClipper needs at least one tensor')
        self.device = self.tensors[0].device
        if self.device.type != 'cuda':
            raise RuntimeError('trebi_amd clips gradients on an MI355X only; there is no CPU path')
        n = len(self.tensors)
        for i, t in enumerate(self.tensors):
            if t.device != self.device:
                raise RuntimeError(f'tensor {i} is on {t.device}, the first one on {self.device}')
            if t.dtype not in _DTYPES:
                raise TypeError(f'tensor {i} has type {t.dtype}; float32, bfloat16 and float16 are supported')
            if not t.is_contiguous():
                raise RuntimeError(f'tensor {i} is not contiguous')
        ptrs = (C.c_void_p * n)(*[t.data_ptr() or None for t in self.tensors])
        numels = (C.c_int64 * n)(*[t.numel() for t in self.tensors])
        dtypes = (C.c_int * n)(*[_DTYPES[t.dtype] for t in self.tensors])
        lib = _lib.lib()
        nbytes = lib.trebi_grad_set_bytes(n, numels)
        host = torch.empty(max(nbytes, 1), dtype=torch.uint8, device='cpu')
        self.set = _lib.GradSet()
        _lib.check(lib.trebi_grad_set_fill(n, ptrs, numels, dtypes, _lib.ptr(host), nbytes, C.byref(self.set)))
        self.table = host.to(self.device)
        self._made_on = _lib.stream(self.device)
        self._spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self.tensors]
        self.total = int(self.set.total)
        self._ws_bytes = lib.trebi_grad_workspace_bytes(C.byref(self.set))
        self._fixed = (_lib.ctx(self.device.index or 0), C.byref(self.set), C.c_void_p(self.table.data_ptr()), self.norm_type)

    def _buffers(self):
        """A workspace of this call's own (two calls may run at once), the norm, the stream."""
        ws, st = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device), _lib.stream(self.device)
        if st != self._made_on:                             # the table's memory waits for this stream before it serves others
            self.table.record_stream(torch.cuda.current_stream(self.device))
        return ws, torch.empty((), dtype=torch.float32, device=self.device), st

    def norm(self, grad_scale=1.0):
        """grad_scale * the norm, a device scalar."""
        ws, norm, st = self._buffers()
        _lib.check(_lib.lib().trebi_grad_norm(*self._fixed, grad_scale, norm.data_ptr(), ws.data_ptr(), self._ws_bytes, st))
        return norm

    def clip_(self, max_norm, grad_scale=1.0):
        """Scale the gradients in place; the norm before clipping."""
        ws, norm, st = self._buffers()
        _lib.check(_lib.lib().trebi_grad_clip(*self._fixed, max_norm, grad_scale, None, norm.data_ptr(), ws.data_ptr(),
                                              self._ws_bytes, st))
        return norm

    def clip_into(self, max_norm, grad_scale=1.0, out=None):
        """(flat, norm): the scaled gradients as one float32 tensor in the tensors' order; the gradients keep their values."""
        if out is None:
            out = torch.empty(self.total, dtype=torch.float32, device=self.device)
        elif out.shape != (self.total,) or out.dtype != torch.float32 or out.device != self.device or not out.is_contiguous():
            raise RuntimeError(f'out must be a contiguous float32 [{self.total}] on {self.device}')
        else:
            lo, hi = out.data_ptr(), out.data_ptr() + 4 * self.total
            for i, (a, b) in enumerate(self._spans):
                if a < hi and lo < b:
                    raise RuntimeError(f'out overlaps tensor {i}; use clip_ to scale in place')
        ws, norm, st = self._buffers()
        _lib.check(_lib.lib().trebi_grad_clip(*self._fixed, max_norm, grad_scale, out.data_ptr() or ws.data_ptr(),
                                              norm.data_ptr(), ws.data_ptr(), self._ws_bytes, st))
        return out, norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for one call: clips the .grad of `parameters` in place and returns their norm.  Waits for the
    copy of the table, with error_if_nonfinite for the norm too; a program that clips every step keeps a GradClipper instead."""
    if torch.is_tensor(parameters):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0, dtype=torch.float32, device='cpu')
    clipper = GradClipper(grads, norm_type)
    if error_if_nonfinite:
        norm = clipper.norm()
        if not torch.isfinite(norm):
            raise RuntimeError(f'the gradient norm is {norm.item()}, nothing was clipped')
    return clipper.clip_(max_norm)
