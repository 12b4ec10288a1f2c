"""A gated linear layer: two linear layers of one input, one of them the other's gate,

    output = act(input Wg + bg) * (input Wu + bu)

with act one of "sigmoid", "silu" (g sigmoid(g)), "gelu" (g Phi(g), Phi the normal distribution's) and "tanh".  The reference has no layer with
two inputs to a product; the names follow its `Model` trait (deep_rl/model/model.mojo:200-273).  A Linear behind it makes a feed-forward block.

Parameters are laid out like those of a Linear(in_dim, 2 * out_dim), [W (in x 2 out, row-major) | b], the gate's columns first, so that
initialisers and optimisers (Adam, and Muon for a model of that Linear) serve as they are.  Rows are [rows, dim] tensors, float32 or bfloat16,
elements of a row next to each other and rows at any equal distance; params have the rows' type (in bfloat16 a copy of the parameters that
the optimiser keeps), gradients of parameters are float32.  In bfloat16 sums are float32 and rounded where they are stored; the gradients of
gate and up, which are not stored, go into that of the input with 16 bits.
"""
import ctypes as C

import torch

from . import _lib
from .context import _on_device, _rows, _scratch

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_ACTIVATIONS = {"sigmoid": 0, "silu": 1, "gelu": 2, "tanh": 3}


class GatedLinear:
    def __init__(self, in_dim, out_dim, activation="silu"):
        if not (1 <= in_dim <= 1 << 16 and 1 <= out_dim <= 1 << 16):
            raise _lib.MrlError("GatedLinear: dims %d and %d: 1 to 65536 expected" % (in_dim, out_dim))
        if activation not in _ACTIVATIONS:
            raise _lib.MrlError("GatedLinear: unknown activation %r: one of %s expected" % (activation, ", ".join(_ACTIVATIONS)))
        self.IN_DIM, self.OUT_DIM, self.PARAM_SIZE, self.activation = in_dim, out_dim, 2 * out_dim * (in_dim + 1), activation
        self._act = _ACTIVATIONS[activation]
        self._sizes = {}   # (device, type, rows, backward) -> workspace bytes

    def _shape(self, name, t):
        if t.dim() != 2:
            raise _lib.MrlError("%s: [rows, %d] expected, got %s" % (name, self.IN_DIM, list(t.shape)))
        kind = _TYPES.get(t.dtype)
        if kind is None:
            raise _lib.MrlError("%s: float32 or bfloat16 expected, got %s" % (name, t.dtype))
        if t.size(0) >= 1 << 26:
            raise _lib.MrlError("%s: %d rows: fewer than 2^26 expected" % (name, t.size(0)))
        return t.size(0), kind

    def _flat(self, ctx, name, t, dtype):
        if t.dtype is not dtype or t.numel() != self.PARAM_SIZE or not t.is_contiguous():
            raise _lib.MrlError("%s: %d contiguous values of %s expected, got %s of %s" % (name, self.PARAM_SIZE, dtype, list(t.shape), t.dtype))
        if t.device != ctx.device:
            _on_device(ctx, name, t)
        return t.data_ptr()

    def _workspace(self, ctx, kind, rows, backward):
        """(tensor or None, pointer, bytes)"""
        key = (ctx.device, kind, rows, backward)
        n = self._sizes.get(key)
        if n is None:
            size = C.c_uint64(0)
            _lib.call("mrl_gated_linear_workspace", ctx.handle, kind, rows, self.IN_DIM, self.OUT_DIM, int(backward), C.byref(size))
            n = self._sizes[key] = size.value
        if n == 0:
            return None, None, 0
        ws = _scratch(ctx, n)
        return ws, ws.data_ptr(), n

    def forward_gpu(self, ctx, output, input, params):
        rows, kind = self._shape("input", input)
        x, x_ld = _rows(ctx, "input", input, (rows, self.IN_DIM), input.dtype)
        o, o_ld = _rows(ctx, "output", output, (rows, self.OUT_DIM), input.dtype)
        p = self._flat(ctx, "params", params, input.dtype)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, kind, rows, False)
        _lib.call("mrl_gated_linear_forward", ctx.handle, kind, self._act, rows, self.IN_DIM, self.OUT_DIM, x, x_ld, p, o, o_ld, ws_ptr, ws_bytes)

    def backward_gpu(self, ctx, grad_input, grads, grad_output, input, params):
        """Overwrites grads (float32, laid out like params) and grad_input (None: not wanted) from the gradient of the output."""
        rows, kind = self._shape("input", input)
        x, x_ld = _rows(ctx, "input", input, (rows, self.IN_DIM), input.dtype)
        g, g_ld = _rows(ctx, "grad_output", grad_output, (rows, self.OUT_DIM), input.dtype)
        gx, gx_ld = (None, 0) if grad_input is None else _rows(ctx, "grad_input", grad_input, (rows, self.IN_DIM), input.dtype)
        p, gp = self._flat(ctx, "params", params, input.dtype), self._flat(ctx, "grads", grads, torch.float32)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, kind, rows, True)
        _lib.call("mrl_gated_linear_backward", ctx.handle, kind, self._act, rows, self.IN_DIM, self.OUT_DIM, g, g_ld, x, x_ld, p, gx, gx_ld, gp,
                  ws_ptr, ws_bytes)
