"""A recurrent layer over time-major rollouts: the gated linear recurrence

    a = sigmoid(gate),   h[t] = a[t] * h[t-1] + (1 - a[t]) * value[t]

with the state cut where an episode ended.  It has no parameters of its own: gate and value are what layers in front of it make
(one Linear(in, 2 * width), whose output rows hold both, say), and its output rows go into the layers behind it.  The
reference has no layer with a state; the names follow its `Model` trait (deep_rl/model/model.mojo:200-273).

Rows are the rollout's (row = t * envs + env): gate, value, output and their gradients are [steps * envs, width] tensors, float32 or
bfloat16, elements of a row next to each other and rows at any equal distance, so that `pre[:, :width]` and `pre[:, width:]` serve
as they are.  States are float32 [envs, width].  `dones` are the rollout's own flags (RolloutBuffers.r_dones), `prev_dones` those
of the step ahead of the first one: where a flag is above 0.5 the next step starts from a zero state.

What a call writes lies apart from what it reads, but for the states that are named below: MrlError where an element of an output
is one of an input or of another output.
"""
import ctypes as C

import torch

from . import _lib
from .context import _on_device, _scratch

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class GatedRecurrence:
    def __init__(self, width):
        if width < 1:
            raise _lib.MrlError("GatedRecurrence: the width must be positive, got %d" % width)
        self.width = width
        self._sizes = {}   # (device, steps, envs) -> workspace bytes

    def _rows(self, ctx, name, t, size, dtype):
        """(pointer, elements from a row to the next) of a tensor of size (rows, width)."""
        if t.shape == size and t.dtype is dtype and t.device == ctx.device:
            row, element = t.stride()
            if element == 1 and row >= size[1]:
                return t.data_ptr(), row
        if t.shape != size:
            raise _lib.MrlError("%s: a [%d, %d] tensor expected, got %s" % (name, *size, list(t.shape)))
        if t.dtype != dtype:
            raise _lib.MrlError("%s: %s expected, got %s" % (name, dtype, t.dtype))
        _on_device(ctx, name, t)
        row, element = t.stride()
        if size[1] > 1 and element != 1 and size[0] > 0:
            raise _lib.MrlError("%s: the elements of a row must be next to each other, got strides %s" % (name, t.stride()))
        if size[0] < 2:
            row = size[1]
        elif row < size[1]:
            raise _lib.MrlError("%s: rows overlap, got strides %s" % (name, t.stride()))
        return t.data_ptr(), row

    def _flat(self, ctx, name, t, n):
        if t is None:
            return None
        if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
            raise _lib.MrlError("%s: %d contiguous floats expected, got %s of %s" % (name, n, list(t.shape), t.dtype))
        if t.device != ctx.device:
            _on_device(ctx, name, t)
        return t.data_ptr()

    def _shape(self, gate, steps):
        if steps < 1 or gate.dim() != 2 or gate.size(0) % steps:
            raise _lib.MrlError("gate: [steps * envs, %d] rows of %d steps expected, got %s" % (self.width, steps, list(gate.shape)))
        kind = _TYPES.get(gate.dtype)
        if kind is None:
            raise _lib.MrlError("gate: float32 or bfloat16 expected, got %s" % gate.dtype)
        if steps >= 1 << 31 or gate.size(0) // steps * self.width >= 1 << 31:
            raise _lib.MrlError("gate: %s of %d steps: fewer than 2^31 steps and states expected" % (list(gate.shape), steps))
        return gate.size(0) // steps, kind

    def _workspace(self, ctx, steps, envs):
        """(tensor or None, pointer, bytes)"""
        if steps == 1:
            return None, None, 0
        key = (ctx.device, steps, envs)
        n = self._sizes.get(key)
        if n is None:
            size = C.c_uint64(0)
            _lib.call("mrl_recurrence_workspace", ctx.handle, steps, envs, self.width, C.byref(size))
            n = self._sizes[key] = size.value
        if n == 0:
            return None, None, 0
        ws = _scratch(ctx, n)
        return ws, ws.data_ptr(), n

    def forward_gpu(self, ctx, output, gate, value, steps, state_in=None, state_out=None, dones=None, prev_dones=None):
        """output and state_out (None: not wanted; may be state_in) from gate, value and state_in (None: zeros)."""
        envs, dtype = self._shape(gate, steps)
        rows, states = steps * envs, envs * self.width
        size, kind = (rows, self.width), gate.dtype
        g, g_ld = self._rows(ctx, "gate", gate, size, kind)
        v, v_ld = self._rows(ctx, "value", value, size, kind)
        o, o_ld = self._rows(ctx, "output", output, size, kind)
        flags, before = self._flat(ctx, "dones", dones, rows), self._flat(ctx, "prev_dones", prev_dones, envs)
        s_in = self._flat(ctx, "state_in", state_in, states)
        s_out = s_in if state_out is state_in else self._flat(ctx, "state_out", state_out, states)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, steps, envs)
        _lib.call("mrl_recurrence_forward", ctx.handle, dtype, steps, envs, self.width, g, g_ld, v, v_ld, flags, before, s_in, o, o_ld,
                  s_out, ws_ptr, ws_bytes)

    def step_gpu(self, ctx, output, gate, value, state, prev_dones=None):
        """One step of every environment, `state` updated in place; prev_dones: the flags of the step before this one."""
        self.forward_gpu(ctx, output, gate, value, 1, state_in=state, state_out=state, prev_dones=prev_dones)

    def backward_gpu(self, ctx, grad_gate, grad_value, grad_output, gate, value, output, steps, state_in=None, dones=None,
                     prev_dones=None, grad_state_out=None, grad_state_in=None):
        """Overwrites grad_gate, grad_value and grad_state_in (None: not wanted; may be grad_state_out) with the gradients of what
        forward_gpu computed, from those of its output and (None: zeros) of state_out."""
        envs, dtype = self._shape(gate, steps)
        rows, states = steps * envs, envs * self.width
        size, kind = (rows, self.width), gate.dtype
        g, g_ld = self._rows(ctx, "gate", gate, size, kind)
        v, v_ld = self._rows(ctx, "value", value, size, kind)
        o, o_ld = self._rows(ctx, "output", output, size, kind)
        go, go_ld = self._rows(ctx, "grad_output", grad_output, size, kind)
        gg, gg_ld = self._rows(ctx, "grad_gate", grad_gate, size, kind)
        gv, gv_ld = self._rows(ctx, "grad_value", grad_value, size, kind)
        flags, before = self._flat(ctx, "dones", dones, rows), self._flat(ctx, "prev_dones", prev_dones, envs)
        s_in = self._flat(ctx, "state_in", state_in, states)
        gs_out, gs_in = self._flat(ctx, "grad_state_out", grad_state_out, states), self._flat(ctx, "grad_state_in", grad_state_in, states)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, steps, envs)
        _lib.call("mrl_recurrence_backward", ctx.handle, dtype, steps, envs, self.width, g, g_ld, v, v_ld, o, o_ld, flags, before, s_in,
                  go, go_ld, gs_out, gg, gg_ld, gv, gv_ld, gs_in, ws_ptr, ws_bytes)
