"""Recurrent layers over time-major rollouts.  GatedRecurrence is the gated linear recurrence

    a = sigmoid(gate),   h[t] = a[t] * h[t-1] + (1 - a[t]) * value[t]

with the state cut where an episode ended.  It has no parameters of its own: gate and value are what layers in front of it make
(one Linear(in, 2 * width), whose output rows hold both, say), and its output rows go into the layers behind it.  The
reference has no layer with a state; the names follow its `Model` trait (deep_rl/model/model.mojo:200-273).

Rows are the rollout's (row = t * envs + env): gate, value, output and their gradients are [steps * envs, width] tensors, float32 or
bfloat16, elements of a row next to each other and rows at any equal distance, so that `pre[:, :width]` and `pre[:, width:]` serve
as they are.  States are float32 [envs, width].  `dones` are the rollout's own flags (RolloutBuffers.r_dones), `prev_dones` those
of the step ahead of the first one: where a flag is above 0.5 the next step starts from a zero state.

GatedDeltaRule has a matrix for a memory: see the class.  Rows, states, flags and cuts are the same.

What a call writes lies apart from what it reads, but for the states that are named below: MrlError where an element of an output
is one of an input or of another output.
"""
import ctypes as C

import torch

from . import _lib
from .context import _on_device, _rows, _scratch

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _flat(ctx, name, t, n):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
        raise _lib.MrlError("%s: %d contiguous floats expected, got %s of %s" % (name, n, list(t.shape), t.dtype))
    if t.device != ctx.device:
        _on_device(ctx, name, t)
    return t.data_ptr()


class GatedRecurrence:
    def __init__(self, width):
        if width < 1:
            raise _lib.MrlError("GatedRecurrence: the width must be positive, got %d" % width)
        self.width = width
        self._sizes = {}   # (device, steps, envs) -> workspace bytes

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
        g, g_ld = _rows(ctx, "gate", gate, size, kind)
        v, v_ld = _rows(ctx, "value", value, size, kind)
        o, o_ld = _rows(ctx, "output", output, size, kind)
        flags, before = _flat(ctx, "dones", dones, rows), _flat(ctx, "prev_dones", prev_dones, envs)
        s_in = _flat(ctx, "state_in", state_in, states)
        s_out = s_in if state_out is state_in else _flat(ctx, "state_out", state_out, states)
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
        g, g_ld = _rows(ctx, "gate", gate, size, kind)
        v, v_ld = _rows(ctx, "value", value, size, kind)
        o, o_ld = _rows(ctx, "output", output, size, kind)
        go, go_ld = _rows(ctx, "grad_output", grad_output, size, kind)
        gg, gg_ld = _rows(ctx, "grad_gate", grad_gate, size, kind)
        gv, gv_ld = _rows(ctx, "grad_value", grad_value, size, kind)
        flags, before = _flat(ctx, "dones", dones, rows), _flat(ctx, "prev_dones", prev_dones, envs)
        s_in = _flat(ctx, "state_in", state_in, states)
        gs_out, gs_in = _flat(ctx, "grad_state_out", grad_state_out, states), _flat(ctx, "grad_state_in", grad_state_in, states)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, steps, envs)
        _lib.call("mrl_recurrence_backward", ctx.handle, dtype, steps, envs, self.width, g, g_ld, v, v_ld, o, o_ld, flags, before, s_in,
                  go, go_ld, gs_out, gg, gg_ld, gv, gv_ld, gs_in, ws_ptr, ws_bytes)


class GatedDeltaRule:
    """The gated delta rule: every head has a memory S [key_dim, value_dim] that maps keys to values,

        a = sigmoid(gate), b = sigmoid(rate), k = key / |key|, q = query / (|query| sqrt(key_dim)), |x| = sqrt(sum x^2 + 1e-6),
        S' = a[t] S[t-1],  S[t] = S' + b[t] k[t] (value[t] - S'^T k[t])^T,  output[t] = S[t]^T q[t].

    Rows are [steps * envs, width] tensors as above: query and key of width key_heads * key_dim, value and output of heads * value_dim,
    gate and rate of heads; heads h of a group of heads / key_heads share a query and a key.  All five can be columns of one Linear's
    output.  States are float32, envs * heads * key_dim * value_dim values in this order."""

    def __init__(self, heads, key_dim, value_dim, key_heads=None):
        key_heads = heads if key_heads is None else key_heads
        if heads < 1 or key_heads < 1 or heads % key_heads:
            raise _lib.MrlError("GatedDeltaRule: %d heads on %d key heads" % (heads, key_heads))
        if not (1 <= key_dim <= 128 and 1 <= value_dim <= 128):
            raise _lib.MrlError("GatedDeltaRule: key_dim %d and value_dim %d: 1 to 128 expected" % (key_dim, value_dim))
        self.heads, self.key_heads, self.key_dim, self.value_dim = heads, key_heads, key_dim, value_dim
        self.key_width, self.value_width, self.state_size = key_heads * key_dim, heads * value_dim, heads * key_dim * value_dim
        self._sizes = {}   # (device, type, steps, envs, backward) -> workspace bytes

    def _describe(self, ctx, query, key, value, gate, rate, steps, state_in, dones, prev_dones):
        """(description, envs, rows, type)"""
        if steps < 1 or value.dim() != 2 or value.size(0) % steps:
            raise _lib.MrlError("value: [steps * envs, %d] rows of %d steps expected, got %s" % (self.value_width, steps, list(value.shape)))
        dtype = value.dtype
        kind = _TYPES.get(dtype)
        if kind is None:
            raise _lib.MrlError("value: float32 or bfloat16 expected, got %s" % dtype)
        rows = value.size(0)
        envs = rows // steps
        if steps >= 1 << 30 or envs * self.heads >= 1 << 22:
            raise _lib.MrlError("value: %s of %d steps: fewer than 2^30 steps and 2^22 heads of environments expected" % (list(value.shape), steps))
        q, q_ld = _rows(ctx, "query", query, (rows, self.key_width), dtype)
        k, k_ld = _rows(ctx, "key", key, (rows, self.key_width), dtype)
        v, v_ld = _rows(ctx, "value", value, (rows, self.value_width), dtype)
        g, g_ld = _rows(ctx, "gate", gate, (rows, self.heads), dtype)
        r, r_ld = _rows(ctx, "rate", rate, (rows, self.heads), dtype)
        return _lib.Delta(kind, steps, envs, self.heads, self.key_heads, self.key_dim, self.value_dim, q, k, v, g, r, q_ld, k_ld, v_ld, g_ld,
                          r_ld, _flat(ctx, "dones", dones, rows), _flat(ctx, "prev_dones", prev_dones, envs),
                          _flat(ctx, "state_in", state_in, envs * self.state_size)), envs, rows, dtype

    def _workspace(self, ctx, d, backward):
        """(tensor or None, pointer, bytes)"""
        key = (ctx.device, d.dtype, d.T, d.N, backward)
        n = self._sizes.get(key)
        if n is None:
            size = C.c_uint64(0)
            _lib.call("mrl_delta_workspace", ctx.handle, C.byref(d), int(backward), C.byref(size))
            n = self._sizes[key] = size.value
        if n == 0:
            return None, None, 0
        ws = _scratch(ctx, n)
        return ws, ws.data_ptr(), n

    def forward_gpu(self, ctx, output, query, key, value, gate, rate, steps, state_in=None, state_out=None, dones=None, prev_dones=None):
        """output and state_out (None: not wanted; may be state_in) from the rows and state_in (None: zeros)."""
        d, envs, rows, dtype = self._describe(ctx, query, key, value, gate, rate, steps, state_in, dones, prev_dones)
        o, o_ld = _rows(ctx, "output", output, (rows, self.value_width), dtype)
        s_out = d.state_in if state_out is state_in else _flat(ctx, "state_out", state_out, envs * self.state_size)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, d, False)
        _lib.call("mrl_delta_forward", ctx.handle, C.byref(d), o, o_ld, s_out, ws_ptr, ws_bytes)

    def step_gpu(self, ctx, output, query, key, value, gate, rate, state, prev_dones=None):
        """One step of every environment, `state` updated in place; prev_dones: the flags of the step before this one."""
        self.forward_gpu(ctx, output, query, key, value, gate, rate, 1, state_in=state, state_out=state, prev_dones=prev_dones)

    def backward_gpu(self, ctx, grad_query, grad_key, grad_value, grad_gate, grad_rate, grad_output, query, key, value, gate, rate, steps,
                     state_in=None, dones=None, prev_dones=None, grad_state_out=None, grad_state_in=None):
        """Overwrites the gradients of the rows and grad_state_in (None: not wanted; may be grad_state_out) with those of what forward_gpu
        computed, from those of its output and (None: zeros) of state_out."""
        d, envs, rows, dtype = self._describe(ctx, query, key, value, gate, rate, steps, state_in, dones, prev_dones)
        o, o_ld = _rows(ctx, "grad_output", grad_output, (rows, self.value_width), dtype)
        q, q_ld = _rows(ctx, "grad_query", grad_query, (rows, self.key_width), dtype)
        k, k_ld = _rows(ctx, "grad_key", grad_key, (rows, self.key_width), dtype)
        v, v_ld = _rows(ctx, "grad_value", grad_value, (rows, self.value_width), dtype)
        g, g_ld = _rows(ctx, "grad_gate", grad_gate, (rows, self.heads), dtype)
        r, r_ld = _rows(ctx, "grad_rate", grad_rate, (rows, self.heads), dtype)
        states = envs * self.state_size
        s_out, s_in = _flat(ctx, "grad_state_out", grad_state_out, states), _flat(ctx, "grad_state_in", grad_state_in, states)
        grads = _lib.DeltaGrads(q, k, v, g, r, q_ld, k_ld, v_ld, g_ld, r_ld, s_in)
        ws, ws_ptr, ws_bytes = self._workspace(ctx, d, True)
        _lib.call("mrl_delta_backward", ctx.handle, C.byref(d), o, o_ld, s_out, C.byref(grads), ws_ptr, ws_bytes)
