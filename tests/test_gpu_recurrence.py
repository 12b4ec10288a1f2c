"""GatedRecurrence against the recurrence and its gradient in 64 bits, step by step."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24      # half a step of fp32, relative
# Roundings that one step adds, in units of the sum of its terms' magnitudes: the exponential and the reciprocal are off by a step
# each (2 units); sigmoid: 4 of the exponential, the sum 1, the reciprocal 2, the product of the smaller side 1 and once more what its
# factor is off: at most 10; the product with the value 1, the multiply-add 1.  1 / ln 2 is kept in one fp32 constant, 0.22 units off,
# which is 0.22 |gate| units of the exponential: the gates here are below 16, so 4 more.  In bf16 the exponential's argument is rounded
# without being corrected, |gate| units of the exponential, 16 more.  A step's share of a composed (A, B) is off by as much again, so
# a state that went through one is off by twice that.
STEP = {"f32": 32 * UNIT, "bf16": 64 * UNIT}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": UNIT, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


def forward64(gate, value, cut, h, step=STEP["f32"]):
    """(states, what they may be off by): [T, N, D] in 64 bits; cut [T, N]: the state ahead of the step counts as 0."""
    a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    off, states, offs = torch.zeros_like(h), [], []
    for t in range(len(gate)):
        c = cut[t][:, None]
        h, off = torch.where(c, torch.zeros_like(h), h), torch.where(c, torch.zeros_like(h), off)
        b = rest[t] * value[t]
        off = a[t] * off + step * (a[t] * h.abs() + b.abs())
        h = a[t] * h + b
        states.append(h)
        offs.append(off)
    return torch.stack(states), torch.stack(offs)


def backward64(gate, value, out, cut, h, grad_out, grad_last, step):
    """(dgate, dvalue, dstate) and what they may be off by."""
    a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    g, off = grad_last, torch.zeros_like(grad_last)
    dg, dx, og, ox = [torch.zeros_like(gate) for _ in range(4)]
    for t in range(len(gate) - 1, -1, -1):
        c = cut[t][:, None]
        before = torch.where(c, torch.zeros_like(h), out[t - 1] if t else h)
        d = grad_out[t] + g
        off = off + UNIT * d.abs()
        dx[t], ox[t] = rest[t] * d, rest[t] * (off + step / 2 * d.abs())
        dg[t] = a[t] * rest[t] * (before - value[t]) * d
        og[t] = a[t] * rest[t] * (before.abs() + value[t].abs()) * (off + step * d.abs())
        g, off = a[t] * d, a[t] * off + step * a[t] * (grad_out[t].abs() + g.abs())
        g, off = torch.where(c, torch.zeros_like(g), g), torch.where(c, torch.zeros_like(g), off)
    return (dg, dx, g), (og, ox, off)


class Case:
    """Inputs on the device, and in 64 bits on the host."""

    def __init__(self, T, N, D, dtype, packed=False, dones=True, state=True, seed=0, rate=0.05):
        gen = torch.Generator().manual_seed(seed + 1000 * T + 100 * N + D)
        self.T, self.N, self.D, self.dtype = T, N, D, dtype
        tt = TYPES[dtype]
        gate = torch.randn(T * N, D, generator=gen) * 2 + torch.linspace(-1, 5, D)
        value = torch.randn(T * N, D, generator=gen)
        if packed:
            pre = torch.cat((gate, value), 1).to(tt).cuda()
            self.gate, self.value = pre[:, :D], pre[:, D:]
        else:
            self.gate, self.value = gate.to(tt).cuda(), value.to(tt).cuda()
        self.state = torch.randn(N, D, generator=gen).cuda() if state else None
        flags = (torch.rand(T + 1, N, generator=gen) < rate).float()
        self.prev, self.dones = (flags[0].cuda(), flags[1:].contiguous().cuda()) if dones else (None, None)
        self.cut = flags[:-1] > 0.5 if dones else torch.zeros(T, N, dtype=torch.bool)
        self.grad_out = torch.randn(T * N, D, generator=gen).to(tt).cuda()
        self.grad_last = torch.randn(N, D, generator=gen).cuda() if state else None

    def host(self, x, *shape):
        return (torch.zeros(*shape) if x is None else x.cpu()).double().reshape(shape)

    def shape(self):
        return self.T, self.N, self.D

    def forward64(self):
        return forward64(self.host(self.gate, *self.shape()), self.host(self.value, *self.shape()), self.cut, self.host(self.state, self.N, self.D),
                         STEP[self.dtype])

    def backward64(self, out):
        return backward64(self.host(self.gate, *self.shape()), self.host(self.value, *self.shape()), self.host(out, *self.shape()), self.cut,
                          self.host(self.state, self.N, self.D), self.host(self.grad_out, *self.shape()), self.host(self.grad_last, self.N, self.D), STEP[self.dtype])

    def forward(self, mrl, ctx):
        out = torch.full((self.T * self.N, self.D), 7.0, dtype=TYPES[self.dtype], device="cuda")
        last = torch.full((self.N, self.D), 7.0, device="cuda")
        mrl.GatedRecurrence(self.D).forward_gpu(ctx, out, self.gate, self.value, self.T, state_in=self.state, state_out=last, dones=self.dones,
                                                prev_dones=self.prev)
        return out, last

    def backward(self, mrl, ctx, out):
        dg, dx = (torch.full((self.T * self.N, self.D), 7.0, dtype=TYPES[self.dtype], device="cuda") for _ in range(2))
        ds = torch.full((self.N, self.D), 7.0, device="cuda")
        mrl.GatedRecurrence(self.D).backward_gpu(ctx, dg, dx, self.grad_out, self.gate, self.value, out, self.T, state_in=self.state,
                                                 dones=self.dones, prev_dones=self.prev, grad_state_out=self.grad_last, grad_state_in=ds)
        return dg, dx, ds


def near(got, want, off, half, what):
    got, off = got.cpu().double().reshape(want.shape), off + half * (want.abs() + off)
    worst = ((got - want).abs() - off).max().item() if want.numel() else -1.0
    assert worst <= 1e-37, "%s: %g beyond its bound at %s" % (what, worst, ((got - want).abs() - off).argmax().item())


# one wavefront per group of channels, workgroups of 2 to 16 wavefronts, segments; widths below a vector, odd ones, a ragged last
# group; steps below, at and one past a tile
SHAPES = [(1, 1, 1), (1, 7, 3), (1, 5, 4), (2, 5, 2), (3, 2, 5), (4, 1, 64), (5, 3, 45), (8, 70, 33), (17, 1, 65), (31, 700, 6), (64, 9, 33),
          (65, 16, 100), (64, 64, 64), (9, 2100, 256), (257, 3, 7), (256, 2, 256), (1000, 2, 250), (4097, 3, 45), (5000, 2, 3), (16384, 1, 64), (255, 3, 40), (300, 40, 36), (256, 1, 1),
          (1023, 5, 17), (260, 600, 250), (140, 40, 200), (150, 70, 255), (600, 130, 64), (520, 300, 3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,D", SHAPES)
def test_forward_and_backward(mrl, ctx, T, N, D, dtype):
    print("recurrence", T, N, D, dtype, flush=True)
    c = Case(T, N, D, dtype, packed=(T + N + D) % 2 == 0, dones=(T + D) % 3 != 0, state=N % 4 != 3)
    out, last = c.forward(mrl, ctx)
    ctx.synchronize()
    want, off = c.forward64()
    near(out, want, off, HALF[dtype] if dtype == "bf16" else 0.0, "out")
    near(last, want[-1], off[-1], 0.0, "state_out")
    if dtype == "f32":
        assert torch.equal(last, out[-N:])
    dg, dx, ds = c.backward(mrl, ctx, out)
    ctx.synchronize()
    wants, offs = c.backward64(out)
    for got, want, off, what in zip((dg, dx, ds), wants, offs, ("grad_gate", "grad_value", "grad_state_in")):
        near(got, want, off, HALF[dtype] if dtype == "bf16" and what != "grad_state_in" else 0.0, what)
    again = c.backward(mrl, ctx, out)
    ctx.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((dg, dx, ds), again))


@pytest.mark.parametrize("T,N,D", [(1, 3, 8), (40, 3, 8), (40, 600, 260), (3000, 2, 12), (3000, 2, 2)])
def test_what_a_cut_hides_goes_nowhere(mrl, ctx, T, N, D):
    """Infinities and NaN ahead of a cut, in states and in gradients behind it."""
    c = Case(T, N, D, "f32", rate=0.0)
    c.prev[1] = 1.0
    c.state[1] = float("nan")
    c.cut[0, 1] = True
    at = T // 2
    if T > 1:
        bad = torch.tensor([float("inf"), float("nan"), float("-inf"), 3e38] * D)[:D].cuda()
        rows = slice((at - 1) * N, at * N)
        c.value[rows] = bad
        c.dones[at - 1] = 1.0
        c.cut[at] = True
    out, last = c.forward(mrl, ctx)
    ctx.synchronize()
    want, off = c.forward64()
    keep = torch.ones(T, dtype=torch.bool)
    if T > 1:
        keep[at - 1] = False
    got = out.view(T, N, D).cpu()
    near(got[keep], want[keep], off[keep], 0.0, "out")
    assert torch.isfinite(got[keep]).all() and torch.isfinite(last).all()
    if T > 1:     # the steps ahead of a cut take nothing from the gradients behind it
        c = Case(T, N, D, "f32", rate=0.0)
        c.dones[at - 1] = 1.0
        c.cut[at] = True
        c.grad_out.view(T, N, D)[at] = float("nan")
        out, _ = c.forward(mrl, ctx)
        dg, dx, ds = c.backward(mrl, ctx, out)
        ctx.synchronize()
        wants, offs = c.backward64(out)
        near(dx.view(T, N, D)[:at].cpu(), wants[1][:at], offs[1][:at], 0.0, "grad_value")
        near(dg.view(T, N, D)[:at].cpu(), wants[0][:at], offs[0][:at], 0.0, "grad_gate")
        near(ds, wants[2], offs[2], 0.0, "grad_state_in")


@pytest.mark.parametrize("T,N,D", [(128, 256, 256), (2000, 10, 200), (1, 300, 256)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_states_as_close_as_plain_fp32_steps(mrl, ctx, T, N, D, dtype):
    """States and their gradients, fp32 in either type, against a sequence of plain fp32 steps: on average within 1.5 times its distance from
    64 bits (the kernels' steps have as many roundings; a composed step adds its own once more)."""
    c = Case(T, N, D, dtype)
    out, last = c.forward(mrl, ctx)
    _, _, ds = c.backward(mrl, ctx, out)
    ctx.synchronize()
    T, N, D = c.shape()
    gate, value, h, g = (c.host(x, *s).float() for x, s in ((c.gate, (T, N, D)), (c.value, (T, N, D)), (c.state, (N, D)), (c.grad_last, (N, D))))
    a, grad = 1 / (1 + torch.exp(-gate)), c.host(c.grad_out, T, N, D).float()
    for t in range(T):
        h = a[t] * torch.where(c.cut[t][:, None], torch.zeros_like(h), h) + (1 - a[t]) * value[t]
    for t in range(T - 1, -1, -1):
        g = torch.where(c.cut[t][:, None], torch.zeros_like(g), a[t] * (grad[t] + g))
    for got, plain, want, what in ((last, h, c.forward64()[0][-1], "state"), (ds, g, c.backward64(out)[0][2], "gradient")):
        assert (got.cpu().double() - want).norm() <= 1.5 * (plain.double() - want).norm(), what


def test_extreme_gates(mrl, ctx):
    """Closed and open gates, far beyond where the exponential ends, and NaN."""
    inf, nan = float("inf"), float("nan")
    gate = torch.tensor([0.0, -0.0, 88.0, -88.0, 200.0, -200.0, 3e38, -3e38, inf, -inf, 1e-30, nan]).cuda().view(1, -1)
    D = gate.shape[1]
    value, state, out = torch.full((1, D), 2.0).cuda(), torch.full((1, D), 5.0).cuda(), torch.empty(1, D).cuda()
    mrl.GatedRecurrence(D).forward_gpu(ctx, out, gate, value, 1, state_in=state)
    ctx.synchronize()
    a = torch.sigmoid(gate.double().cpu())
    want = a * 5 + (1 - a) * 2
    got = out.double().cpu()
    assert torch.isnan(got[0, -1]) and (got[0, :-1] - want[0, :-1]).abs().max() <= STEP["f32"] * 7


@pytest.mark.parametrize("T,cut_at,N,D,dtype", [(50, 17, 6, 20, "f32"), (2000, 1000, 2, 36, "bf16"), (7, 1, 1500, 130, "f32")])
def test_pieces_give_the_whole(mrl, ctx, T, cut_at, N, D, dtype):
    c = Case(T, N, D, dtype, rate=0.2)
    whole, last = c.forward(mrl, ctx)
    layer, out, state = mrl.GatedRecurrence(D), torch.empty_like(whole), c.state.clone()
    k = cut_at * N
    layer.forward_gpu(ctx, out[:k], c.gate[:k], c.value[:k], cut_at, state_in=state, state_out=state, dones=c.dones[:cut_at], prev_dones=c.prev)
    layer.forward_gpu(ctx, out[k:], c.gate[k:], c.value[k:], T - cut_at, state_in=state, state_out=state, dones=c.dones[cut_at:],
                      prev_dones=c.dones[cut_at - 1])
    ctx.synchronize()
    want, off = c.forward64()
    near(out, want, off, HALF[dtype] if dtype == "bf16" else 0.0, "out")
    near(state, want[-1], off[-1], 0.0, "state_out")


@pytest.mark.parametrize("N,D,dtype", [(1, 64, "bf16"), (16, 5, "f32"), (8192, 256, "f32"), (3, 1, "f32")])
def test_steps_in_place_are_the_scan(mrl, ctx, N, D, dtype):
    T = 5
    c = Case(T, N, D, dtype, rate=0.3, packed=True)
    layer, state = mrl.GatedRecurrence(D), c.state.clone()
    out = torch.empty(T * N, D, dtype=TYPES[dtype], device="cuda")
    for t in range(T):
        rows = slice(t * N, (t + 1) * N)
        layer.step_gpu(ctx, out[rows], c.gate[rows], c.value[rows], state, prev_dones=c.dones[t - 1] if t else c.prev)
    ctx.synchronize()
    want, off = c.forward64()
    near(out, want, off, HALF[dtype] if dtype == "bf16" else 0.0, "out")
    near(state, want[-1], off[-1], 0.0, "state")


@pytest.mark.parametrize("T,N,D", [(6, 4, 7), (300, 2, 6), (3000, 1, 5)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_at_a_distance_and_odd_addresses(mrl, ctx, T, N, D, dtype):
    """Rows inside wider buffers, starting one element in: what lies between them stays."""
    c = Case(T, N, D, dtype)
    want, off = c.forward64()
    tt, half = TYPES[dtype], HALF[dtype] if dtype == "bf16" else 0.0

    def inside(x, ld, at):
        wide = torch.full((T * N, ld), -3.0, dtype=tt, device="cuda")
        if x is not None:
            wide[:, at:at + D] = x
        return wide, wide[:, at:at + D]
    (_, g), (_, v), (wide, out) = inside(c.gate, D + 3, 1), inside(c.value, 2 * D + 1, D + 1), inside(None, D + 5, 3)
    layer = mrl.GatedRecurrence(D)
    layer.forward_gpu(ctx, out, g, v, T, state_in=c.state, dones=c.dones, prev_dones=c.prev)
    ctx.synchronize()
    near(out, want, off, half, "out")
    assert (wide[:, :3] == -3).all() and (wide[:, 3 + D:] == -3).all()
    wants, offs = c.backward64(out.contiguous())
    (wg, dg), (wv, dv), (_, go) = inside(None, D + 2, 1), inside(None, D + 9, 4), inside(c.grad_out, D + 1, 1)
    ds = torch.empty(N, D, device="cuda")
    layer.backward_gpu(ctx, dg, dv, go, g, v, out, T, state_in=c.state, dones=c.dones, prev_dones=c.prev, grad_state_out=c.grad_last, grad_state_in=ds)
    ctx.synchronize()
    near(dg, wants[0], offs[0], half, "grad_gate")
    near(dv, wants[1], offs[1], half, "grad_value")
    near(ds, wants[2], offs[2], 0.0, "grad_state_in")
    assert (wg[:, :1] == -3).all() and (wg[:, 1 + D:] == -3).all() and (wv[:, :4] == -3).all() and (wv[:, 4 + D:] == -3).all()


@pytest.mark.parametrize("T,N,D", [(5, 3, 45), (64, 200, 64), (300, 9, 40), (2000, 2, 52)])
def test_bf16_gradient_is_that_of_the_states_before_rounding(mrl, ctx, T, N, D):
    """The backward pass takes h' from `out`, rounded to bf16: against autograd through the unrounded states in 64 bits, the gate's gradient is off by that
    rounding, half a step of each h', and no more; the others do not depend on it."""
    c = Case(T, N, D, "bf16", rate=0.1)
    out, _ = c.forward(mrl, ctx)
    got = c.backward(mrl, ctx, out)
    ctx.synchronize()
    gate, value, state = (x.requires_grad_() for x in (c.host(c.gate, T, N, D), c.host(c.value, T, N, D), c.host(c.state, N, D)))
    a, h, states = torch.sigmoid(gate), state, []
    for t in range(T):
        h = a[t] * torch.where(c.cut[t][:, None], torch.zeros_like(h), h) + (1 - a[t]) * value[t]
        states.append(h)
    grad, last = c.host(c.grad_out, T, N, D), c.host(c.grad_last, N, D)
    ((torch.stack(states) * grad).sum() + (h * last).sum()).backward()
    wants = gate.grad, value.grad, state.grad
    gate, value, state, a = gate.detach(), value.detach(), state.detach(), a.detach()
    exact, off = c.forward64()
    offs = backward64(gate, value, exact, c.cut, state, grad, last, STEP["bf16"])[1]
    before, behind = torch.cat((torch.zeros(1, N, D), exact[:-1].abs())), torch.cat((torch.zeros(1, N, D), off[:-1]))
    # the gradient's a (1 - a) d h', where (1 - a) d is that of the value
    rounding = (~c.cut)[..., None] * (HALF["bf16"] * (before + behind) + behind) * a * wants[1].abs()
    for x, want, o, what in zip(got, wants, (offs[0] + rounding, offs[1], offs[2]), ("grad_gate", "grad_value", "grad_state_in")):
        near(x, want, o, 0.0 if what == "grad_state_in" else HALF["bf16"], what)


def test_gradient_against_differences(mrl, ctx):
    """Directional derivatives of the recurrence in 64 bits, taken as differences."""
    c = Case(23, 3, 10, "f32", rate=0.1)
    out, _ = c.forward(mrl, ctx)
    dg, dx, ds = c.backward(mrl, ctx, out)
    ctx.synchronize()
    T, N, D = c.shape()
    gate, value, state = c.host(c.gate, T, N, D), c.host(c.value, T, N, D), c.host(c.state, N, D)
    weights, last = c.host(c.grad_out, T, N, D), c.host(c.grad_last, N, D)

    def loss(g, x, h):
        states = forward64(g, x, c.cut, h)[0]
        return ((states * weights).sum() + (states[-1] * last).sum()).item()
    gen = torch.Generator().manual_seed(5)
    for grad, which in ((dg, 0), (dx, 1), (ds, 2)):
        for _ in range(3):
            at = [gate, value, state]
            v = torch.randn(at[which].shape, generator=gen, dtype=torch.float64)
            eps = 1e-5
            up, down = list(at), list(at)
            up[which], down[which] = at[which] + eps * v, at[which] - eps * v
            want = (loss(*up) - loss(*down)) / (2 * eps)
            terms = grad.cpu().double().reshape(v.shape) * v
            # differences: eps^2 of third derivatives and 2^-52 / eps of the loss's terms; the gradient: fp32 roundings of every term
            # (states are read back in fp32)
            assert abs(terms.sum().item() - want) <= 1e-5 * terms.abs().sum().item() + 1e-8 * (weights.abs().sum().item() + last.abs().sum().item())


def test_other_streams_and_captured_graphs(mrl, ctx):
    """Two graphs of one context's calls, each with a workspace of its own, replayed on different streams with eager calls between."""
    cases = [Case(2000, 2, 40, "f32", seed=s) for s in (1, 2)]
    wants = [c.forward(mrl, ctx) for c in cases]
    grads = [c.backward(mrl, ctx, w[0]) for c, w in zip(cases, wants)]
    ctx.synchronize()
    side = torch.cuda.Stream()
    cctx = mrl.DeviceContext("cuda:0", stream=side)
    graphs, outs = [], []
    for c in cases:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, last = c.forward(mrl, cctx)
            g = c.backward(mrl, cctx, out)
        graphs.append(graph)
        outs.append((out, last, *g))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        cases[0].forward(mrl, ctx)
        torch.cuda.synchronize()
        for o, w, g in zip(outs, wants, grads):
            assert all(torch.equal(x, y) for x, y in zip(o, (*w, *g)))
    del graphs
    cctx.close()


def test_state_goes_through_no_steps_and_no_rows(mrl, ctx):
    lib = mrl._lib.lib()
    a, b = torch.randn(12, device="cuda"), torch.zeros(12, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    assert lib.mrl_recurrence_forward(ctx.handle, 0, 0, 3, 4, None, 0, None, 0, None, None, p(a), None, 0, p(b), None, 0) == 0
    ctx.synchronize()
    assert torch.equal(a, b)
    assert lib.mrl_recurrence_backward(ctx.handle, 1, 0, 3, 4, None, 0, None, 0, None, 0, None, None, None, None, 0, None, None, 0, None, 0,
                                       p(b), None, 0) == 0
    ctx.synchronize()
    assert not b.any()
    layer = mrl.GatedRecurrence(4)
    layer.forward_gpu(ctx, *(torch.empty(0, 4, device="cuda") for _ in range(3)), 5)
    ctx.synchronize()


def test_library_refusals(mrl, ctx):
    lib, x = mrl._lib.lib(), torch.zeros(1 << 16, device="cuda")
    p, size = ctypes.c_void_p(x.data_ptr()), ctypes.c_uint64(0)

    def forward(dtype=0, T=2, N=3, D=4, gate=p, ld=4, ws=None, n=0):
        return lib.mrl_recurrence_forward(ctx.handle, dtype, T, N, D, gate, ld, p, 4, None, None, None, p, 4, None, ws, n)
    for bad, text in ((dict(dtype=2), b"element type"), (dict(T=-1), b"negative"), (dict(N=1 << 20, D=1 << 12), b"2^31"), (dict(gate=None), b"NULL"),
                      (dict(ld=3), b"stride"), (dict(T=4000, N=1), b"workspace holds")):
        assert forward(**bad) == -1 and text in lib.mrl_last_error(), bad
    assert lib.mrl_recurrence_workspace(ctx.handle, 4000, 1, 4, ctypes.byref(size)) == 0 and 0 < size.value <= 1 << 17
    assert forward(T=4000, N=1, ws=p, n=size.value - 1) == -1
    assert forward(T=4000, N=1, ws=ctypes.c_void_p(x.data_ptr() + 4), n=size.value) == -1 and b"aligned" in lib.mrl_last_error()
    assert lib.mrl_recurrence_backward(ctx.handle, 0, 2, 3, 4, p, 4, p, 4, p, 4, None, None, None, p, 4, None, p, 4, None, 4, None, None, 0) == -1
    ctx.synchronize()
    assert not x.any()


def test_outputs_on_inputs_are_refused(mrl, ctx):
    """Before anything is launched: the buffers stay as they are.  Rows between each other are apart."""
    T, N, D = 40, 3, 8
    layer, wide, flat = mrl.GatedRecurrence(D), torch.randn(T * N + N, 5 * D, device="cuda"), torch.randn(4, N, D, device="cuda")
    flags = torch.zeros(T, N, device="cuda")
    gate, value, out, gg, gv = (wide[N:, k * D:(k + 1) * D] for k in range(5))
    before = wide.clone()

    def forward(**other):
        layer.forward_gpu(ctx, **{**dict(output=out, gate=gate, value=value, steps=T, state_in=flat[0], state_out=flat[1], dones=flags), **other})

    def backward(**other):
        layer.backward_gpu(ctx, **{**dict(grad_gate=gg, grad_value=gv, grad_output=grad, gate=gate, value=value, output=out, steps=T, state_in=flat[0], dones=flags,
                                          grad_state_out=flat[2], grad_state_in=flat[3]), **other})
    grad = torch.randn(T * N, D, device="cuda")
    for bad in (dict(output=gate), dict(output=value), dict(output=wide[:-N, D:2 * D]), dict(output=wide[N:, D - 1:2 * D - 1]), dict(output=wide[N:, 2 * D - 1:3 * D - 1]),
                dict(state_out=flat.view(-1)[4:4 + N * D].view(N, D)), dict(dones=wide.view(-1)[-T * N:]), dict(prev_dones=flat[1].view(-1)[:N]),
                dict(state_out=wide.view(-1)[9 * 5 * D:9 * 5 * D + N * D]), dict(state_in=wide.view(-1)[-N * D:])):
        with pytest.raises(mrl.MrlError, match="overlap"):
            forward(**bad)
    for bad in (dict(grad_gate=gate), dict(grad_gate=gv), dict(grad_value=out), dict(grad_value=wide[:-N, 2 * D:3 * D]), dict(grad_output=gv), dict(grad_state_in=flat[0]),
                dict(grad_state_in=grad[-N:]), dict(grad_state_out=flat.view(-1)[3 * N * D - 1:4 * N * D - 1]), dict(grad_gate=grad)):
        with pytest.raises(mrl.MrlError, match="overlap"):
            backward(**bad)
    ctx.synchronize()
    assert torch.equal(wide, before)
    # the same buffers as they may lie, and the states that may be the same
    forward()
    forward(state_out=flat[0])
    backward()
    backward(grad_state_in=flat[2])
    ctx.synchronize()
    assert torch.equal(wide[:, :2 * D], before[:, :2 * D]) and torch.equal(wide[:N], before[:N]) and not torch.equal(wide[N:, 2 * D:], before[N:, 2 * D:])


def test_a_single_row_has_no_distance_to_a_next(mrl, ctx):
    """Whatever is given for it, as one row of a larger buffer may have."""
    lib, x = mrl._lib.lib(), torch.randn(3, 4, device="cuda")
    p = [ctypes.c_void_p(row.data_ptr()) for row in x]
    for ld in (4, 1 << 40, 1 << 62, (1 << 63) - 1):
        assert lib.mrl_recurrence_forward(ctx.handle, 0, 1, 1, 4, p[0], ld, p[1], ld, None, None, None, p[2], ld, None, None, 0) == 0, lib.mrl_last_error()
        ctx.synchronize()
        want = (1 - torch.sigmoid(x[0].double())) * x[1].double()
        assert ((x[2].double() - want).abs() <= STEP["f32"] * want.abs()).all()
        x[2].zero_()
        torch.cuda.synchronize()
        assert lib.mrl_recurrence_forward(ctx.handle, 0, 1, 1, 4, p[0], ld, p[1], ld, None, None, None, p[1], ld, None, None, 0) == -1 and b"overlap" in lib.mrl_last_error()
