"""Optimisers behind the reference's `Optimizer` trait (deep_rl/optimizer/optimizer.mojo:51-68): Adam
(deep_rl/optimizer/adam.mojo) and Muon, which updates a network's hidden matrices by their orthogonalised momentum and everything
else by Adam.  `t` and `lr` live on the host object, as in the reference (the PPO agent anneals `lr` between rollouts); state is
[PARAM_SIZE, 2] interleaved (m, v)."""
import array
import ctypes as C
import functools

import torch

from . import _lib
from .context import _on_device, _ptr, _scratch


class Adam:
    STATE_PER_PARAM = 2

    def __init__(self, lr=0.001, beta1=0.9, beta2=0.999, eps=1e-8):
        self.lr, self.beta1, self.beta2, self.eps, self.t = lr, beta1, beta2, eps, 0

    def step_gpu(self, ctx, params_buf, grads_buf, state_buf):
        n = params_buf.numel()
        if grads_buf.numel() != n or state_buf.numel() != 2 * n:
            raise _lib.MrlError("Adam.step_gpu: grads must hold n and state 2n floats")
        self.t += 1
        _lib.call("mrl_adam_step", ctx.handle, _ptr(params_buf), _ptr(grads_buf), _ptr(state_buf), n,
                  self.t, self.lr, self.beta1, self.beta2, self.eps)


_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def clip_grad_norm(ctx, out, grads, max_norm, norm=None):
    """out[i] = grads[i] * min(1, max_norm / (norm + 1e-8)) with the norm of all values of all tensors, which `norm`, one float32 value, receives
    before clipping (None: not wanted).  grads and out are sequences of contiguous float32 or bfloat16 tensors; out[i] may be grads[i], but
    not overlap a tensor otherwise.  ppo.clip_grad_norm is the same for one vector."""
    if len(out) != len(grads):
        raise _lib.MrlError("clip_grad_norm: %d outputs for %d gradients" % (len(out), len(grads)))
    index = ctx.device.index if ctx.device.type == "cuda" else None   # (an int is compared faster than a device)
    words = []                                                        # a Tensor is four: src, out, n, dtype
    for i, (o, g) in enumerate(zip(out, grads)):
        dtype = g.dtype
        kind = _TYPES.get(dtype)
        if kind is None:
            raise _lib.MrlError("clip_grad_norm: grads[%d]: float32 or bfloat16 expected, got %s" % (i, dtype))
        if not g.is_contiguous():
            raise _lib.MrlError("clip_grad_norm: grads[%d] must be contiguous" % i)
        if g.get_device() != index:
            _on_device(ctx, "grads[%d]" % i, g)
        at = g.data_ptr()
        if o is g:
            words += (at, at, g.numel(), kind)
            continue
        if o.dtype is not dtype or o.shape != g.shape:
            raise _lib.MrlError("clip_grad_norm: out[%d] %s of %s does not fit %s of %s" % (i, list(o.shape), o.dtype, list(g.shape), dtype))
        if not o.is_contiguous():
            raise _lib.MrlError("clip_grad_norm: out[%d] must be contiguous" % i)
        if o.get_device() != index:
            _on_device(ctx, "out[%d]" % i, o)
        words += (at, o.data_ptr(), g.numel(), kind)
    if not max_norm >= 0:
        raise _lib.MrlError("clip_grad_norm: max_norm %s is below 0" % max_norm)
    if norm is not None:
        if norm.numel() != 1 or norm.dtype is not torch.float32:
            raise _lib.MrlError("clip_grad_norm: norm: one float32 value expected, got %s of %s" % (list(norm.shape), norm.dtype))
        _on_device(ctx, "norm", norm)
    ws = _scratch(ctx, _lib.CLIP_TENSORS_WORKSPACE)
    count = len(grads)
    tensors = (_lib.Tensor * count).from_buffer(array.array("q", words)) if count else None
    _lib.call("mrl_clip_tensors", ctx.handle, count, tensors, float(max_norm), None if norm is None else norm.data_ptr(), ws.data_ptr(),
              _lib.CLIP_TENSORS_WORKSPACE)


@functools.lru_cache(maxsize=None)
def _orthogonalize_bytes(count, rows, cols):
    size = C.c_uint64(0)
    _lib.call("mrl_orthogonalize_workspace", count, rows, cols, C.byref(size))
    return size.value


def orthogonalize(ctx, out, x, steps=5, eps=1e-7):
    """out = the Newton-Schulz polynomial of x [rows, cols] or of every matrix of x [count, rows, cols]: x / (|x| + eps), then `steps`
    times X <- 3.4445 X - 4.7750 (X X^T) X + 2.0315 (X X^T)^2 X, which takes the singular values into about [0.7, 1.2].  float32 or
    bfloat16, contiguous; out may be x, but not overlap it otherwise."""
    shape, kind = x.shape, _TYPES.get(x.dtype)
    if len(shape) not in (2, 3) or kind is None:
        raise _lib.MrlError("orthogonalize: a float32 or bfloat16 [rows, cols] or [count, rows, cols] tensor expected, got %s of %s"
                            % (list(shape), x.dtype))
    if out.shape != shape or out.dtype is not x.dtype:
        raise _lib.MrlError("orthogonalize: out %s of %s does not fit x %s of %s" % (list(out.shape), out.dtype, list(shape), x.dtype))
    if x.device != ctx.device or out.device != ctx.device:
        _on_device(ctx, "x", x)
        _on_device(ctx, "out", out)
    if not (x.is_contiguous() and out.is_contiguous()):
        raise _lib.MrlError("orthogonalize: x and out must be contiguous")
    count, rows, cols = shape if len(shape) == 3 else (1, *shape)
    if count * rows * cols == 0:
        return
    if max(count, rows, cols) >= 1 << 31:
        raise _lib.MrlError("orthogonalize: %s is more than the library counts" % list(shape))
    n = _orthogonalize_bytes(count, rows, cols)
    ws = _scratch(ctx, n) if n else None
    _lib.call("mrl_orthogonalize", ctx.handle, kind, count, rows, cols, x.data_ptr(), out.data_ptr(), steps, eps,
              ws.data_ptr() if n else None, n)


class Muon:
    """Momentum, orthogonalised, for the weight matrices of `model`'s hidden layers (all layers but the last, or those numbered in
    `layers`): with a matrix W [in, out], its gradient g and momentum v,

        v <- momentum v + g;   u = g + momentum v (nesterov; else v);   W <- (1 - lr weight_decay) W - lr sqrt(max(1, out / in)) O(u),

    O as in orthogonalize(steps, eps).  Biases and the other layers are updated as by Adam(adam_lr, beta1, beta2, adam_eps).  State is
    Adam's; a matrix's share of it starts with v.  For networks updated by Network.update_gpu: PPOUpdate, and with it the agents,
    apply Adam in kernels of their own and refuse a Muon."""
    STATE_PER_PARAM = 2

    def __init__(self, model, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, eps=1e-7, layers=None, adam_lr=3e-4,
                 beta1=0.9, beta2=0.999, adam_eps=1e-8):
        self.lr, self.momentum, self.nesterov, self.weight_decay, self.steps, self.eps = lr, momentum, nesterov, weight_decay, steps, eps
        self.adam_lr, self.beta1, self.beta2, self.adam_eps, self.t = adam_lr, beta1, beta2, adam_eps, 0
        chosen = range(len(model.layers) - 1) if layers is None else sorted(set(layers))
        if any(not 0 <= k < len(model.layers) for k in chosen):
            raise _lib.MrlError("Muon: layers %s of a model of %d" % (list(chosen), len(model.layers)))
        at, matrices = 0, []
        for k, (kind, rows, cols) in enumerate(model.layers):
            if k in chosen:
                matrices.append(_lib.Matrix(at, rows, cols))
            at += rows * cols + (2 if kind == _lib.STOCHASTIC_ACTOR else 1) * cols
        self._n = model.PARAM_SIZE
        if at != self._n:
            raise _lib.MrlError("Muon: the layers' parameters add up to %d, the model's to %d" % (at, self._n))
        self._matrices = (_lib.Matrix * max(1, len(matrices)))(*matrices)
        self._count = len(matrices)
        size = C.c_uint64(0)
        _lib.call("mrl_muon_workspace", self._count, self._matrices, C.byref(size))
        self._bytes = size.value

    def step_gpu(self, ctx, params_buf, grads_buf, state_buf):
        n = self._n
        for name, t, want in (("params", params_buf, n), ("grads", grads_buf, n), ("state", state_buf, 2 * n)):
            if t.numel() != want or t.dtype is not torch.float32:
                raise _lib.MrlError("Muon.step_gpu: %s must be %d floats, got %d of %s" % (name, want, t.numel(), t.dtype))
            if t.device != ctx.device:
                _on_device(ctx, name, t)
        ws = _scratch(ctx, self._bytes) if self._bytes else None
        _lib.call("mrl_muon_step", ctx.handle, _ptr(params_buf), _ptr(grads_buf), _ptr(state_buf), n, self._count, self._matrices,
                  self.t + 1, self.lr, self.momentum, int(self.nesterov), self.weight_decay, self.steps, self.eps, self.adam_lr, self.beta1,
                  self.beta2, self.adam_eps, ws.data_ptr() if self._bytes else None, self._bytes)
        self.t += 1
