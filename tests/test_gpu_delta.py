"""GatedDeltaRule against the rule and its gradient in 64 bits, step by step."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24      # half a step of fp32, relative
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": UNIT, "bf16": 2.0 ** -8}   # of a stored row; states are fp32
# What values may be off by, of the largest of their head.  The rule is a contraction (|I - b k k^T| <= 1 for 0 <= b <= 1), so what a step
# adds does not grow.  A step's value goes through three sums, over the key's 128, the tile's 16 and once more 16 products, and through
# some ten single roundings in its factors (two sigmoids, lengths, up to 16 products of decays): with independent roundings
# (sqrt(128) + 2 sqrt(16) + 10) units, 30, and a state remembers some tens of steps whose errors add as independent ones do, beside
# values that add the same way.  The gradients go through the same sums twice.
FORWARD, BACKWARD = 64 * UNIT, 160 * UNIT
EPS = 1e-6


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


def rule64(rows, state, cut, heads, key_heads, dk, dv):
    """(outputs [T, N, heads, dv], last state, query and key over their lengths, the lengths) of rows in 64 bits"""
    T, N = cut.shape
    q, k, v, gate, rate = rows
    group = heads // key_heads
    q, k = (x.reshape(T, N, key_heads, dk) for x in (q, k))
    lengths = [(x.square().sum(-1, keepdim=True) + EPS).sqrt() for x in (q, k)]
    q, k = q / lengths[0], k / lengths[1]
    units = q, k
    q, k = (x.repeat_interleave(group, 2) for x in (q / dk ** 0.5, k))
    v = v.reshape(T, N, heads, dv)
    a, b = (torch.sigmoid(x).reshape(T, N, heads, 1, 1) for x in (gate, rate))
    outs = []
    for t in range(T):
        state = torch.where(cut[t].view(N, 1, 1, 1), torch.zeros_like(state), a[t] * state)
        u = b[t] * (v[t].unsqueeze(2) - k[t].unsqueeze(2) @ state)
        state = state + k[t].unsqueeze(3) * u
        outs.append((q[t].unsqueeze(2) @ state).squeeze(2))
    return torch.stack(outs), state, units, lengths


class Case:
    """Inputs on the device, and in 64 bits on the host."""
    NAMES = ("query", "key", "value", "gate", "rate")

    def __init__(self, T, N, heads, key_heads, dk, dv, dtype, packed=False, dones=True, state=True, seed=0, rate=0.05, alike=0.7):
        gen = torch.Generator().manual_seed(seed + 1000 * T + 100 * N + 10 * dk + dv)
        self.T, self.N, self.dtype, self.tt = T, N, dtype, TYPES[dtype]
        self.dims = heads, key_heads, dk, dv
        self.heads, self.dk, self.dv = heads, dk, dv
        self.widths = (key_heads * dk, key_heads * dk, heads * dv, heads, heads)
        rows = [torch.randn(T * N, w, generator=gen) for w in self.widths]
        rows[1] += alike * torch.randn(N, self.widths[1], generator=gen).repeat(T, 1)
        rows[3] = rows[3] * 2 + torch.linspace(-3, 5, heads)
        rows = [x.to(self.tt) for x in rows]
        if packed:
            self.rows = [x for x in torch.cat(rows, 1).cuda().split(self.widths, 1)]
        else:
            self.rows = [x.cuda() for x in rows]
        self.state = torch.randn(N, heads, dk, dv, generator=gen).cuda() if state else None
        flags = (torch.rand(T + 1, N, generator=gen) < rate).float()
        self.prev, self.dones = (flags[0].cuda(), flags[1:].contiguous().cuda()) if dones else (None, None)
        self.cut = flags[:-1] > 0.5 if dones else torch.zeros(T, N, dtype=torch.bool)
        self.grad_out = torch.randn(T * N, heads * dv, generator=gen).to(self.tt).cuda()
        self.grad_last = torch.randn(N, heads, dk, dv, generator=gen).cuda() if state else None

    def layer(self, mrl):
        heads, key_heads, dk, dv = self.dims
        return mrl.GatedDeltaRule(heads, dk, dv, key_heads=key_heads)

    def rows64(self):
        return [x.cpu().double() for x in self.rows]

    def state64(self):
        return torch.zeros(self.N, self.heads, self.dk, self.dv, dtype=torch.float64) if self.state is None else self.state.cpu().double()

    def forward64(self):
        out, last, _, _ = rule64(self.rows64(), self.state64(), self.cut, *self.dims)
        return out.reshape(self.T * self.N, -1), last

    def backward64(self):
        """The gradients of the rows and of the first state, and what roundings in those of query and key are of the size of: with
        n = x / |x|, dx = (dn - n (n dn)) / |x| is a difference of terms up to |dn| / |x|, each rounded, and may be far smaller than they
        are (key_dim 1: dx is 1e-6 / |x|^2 of them)."""
        rows, state = [x.requires_grad_() for x in self.rows64()], self.state64().requires_grad_()
        out, last, units, lengths = rule64(rows, state, self.cut, *self.dims)
        loss = (out.reshape(self.T * self.N, -1) * self.grad_out.cpu().double()).sum()
        if self.grad_last is not None:
            loss = loss + (last * self.grad_last.cpu().double()).sum()
        found = torch.autograd.grad(loss, [*rows, state, *units])
        terms = [(g.norm(dim=-1, keepdim=True) / length).expand_as(g).reshape(self.T * self.N, -1) for g, length in zip(found[6:], lengths)]
        return found[:6], dict(query=terms[0], key=terms[1])

    def forward(self, mrl, ctx, state_out=True):
        out = torch.full((self.T * self.N, self.heads * self.dv), 7.0, dtype=self.tt, device="cuda")
        last = torch.full((self.N, self.heads, self.dk, self.dv), 7.0, device="cuda") if state_out else None
        self.layer(mrl).forward_gpu(ctx, out, *self.rows, self.T, state_in=self.state, state_out=last, dones=self.dones, prev_dones=self.prev)
        return out, last

    def backward(self, mrl, ctx, grad_state=True):
        grads = [torch.full((self.T * self.N, w), 7.0, dtype=self.tt, device="cuda") for w in self.widths]
        first = torch.full((self.N, self.heads, self.dk, self.dv), 7.0, device="cuda") if grad_state else None
        self.layer(mrl).backward_gpu(ctx, *grads, self.grad_out, *self.rows, self.T, state_in=self.state, dones=self.dones, prev_dones=self.prev,
                                     grad_state_out=self.grad_last, grad_state_in=first)
        return [*grads, first]


def near(got, want, heads, off, half, what, size=None):
    """off: of the largest value (of `size`) of the same head; half: of each value"""
    got, size = got.cpu().double().reshape(want.shape), want if size is None else size
    parts = want.shape[0], heads, -1
    if want.dim() == 2:      # rows: [rows, heads * width]
        got, want = got.reshape(parts), want.reshape(parts)
        largest = size.reshape(parts).abs().amax((0, 2), keepdim=True)
    else:                    # states: [N, heads, dk, dv]
        largest = size.abs().amax((0, 2, 3), keepdim=True)
    worst = ((got - want).abs() - off * largest - half * want.abs()).max().item()
    assert worst <= 1e-30, "%s: %g beyond its bound, largest %g" % (what, worst, largest.max().item())


# steps below, at and one past a tile, a block of four (64) and of two (32) tiles; odd dims, dims past 16, 32, 64; groups of heads
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 5, 2, 2, 64, 64), (1, 3, 4, 2, 128, 128), (1, 7, 3, 1, 40, 24), (1, 2, 2, 1, 33, 65), (1, 9, 1, 1, 7, 5),
          (2, 3, 2, 2, 16, 16), (3, 2, 3, 3, 5, 3), (15, 2, 2, 1, 32, 32), (16, 3, 2, 2, 64, 64), (17, 1, 4, 4, 64, 48), (33, 2, 6, 2, 24, 40),
          (64, 2, 2, 2, 64, 64), (65, 3, 2, 1, 128, 128), (32, 1, 1, 1, 128, 16), (33, 2, 2, 2, 100, 17), (130, 2, 3, 1, 40, 24), (129, 1, 2, 2, 17, 128),
          (200, 3, 2, 2, 64, 64), (300, 1, 2, 1, 128, 100), (97, 40, 1, 1, 16, 80), (70, 5, 3, 3, 1, 1),
          # long rollouts of few environments, which go in parts
          (1000, 1, 1, 1, 8, 8), (700, 2, 3, 1, 24, 40), (600, 1, 2, 2, 64, 64), (500, 2, 1, 1, 128, 72), (1030, 3, 1, 1, 40, 128)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,key_heads,dk,dv", SHAPES)
def test_forward(mrl, ctx, T, N, heads, key_heads, dk, dv, dtype):
    print("delta", T, N, heads, key_heads, dk, dv, dtype, flush=True)
    c = Case(T, N, heads, key_heads, dk, dv, dtype, packed=(T + N + dk) % 2 == 0, dones=(T + dk) % 3 != 0, state=N % 4 != 3)
    out, last = c.forward(mrl, ctx)
    ctx.synchronize()
    want, want_last = c.forward64()
    near(out, want, heads, FORWARD, HALF[dtype], "out")
    near(last, want_last, heads, FORWARD, UNIT, "state_out")
    again, _ = c.forward(mrl, ctx, state_out=False)
    ctx.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,key_heads,dk,dv", SHAPES)
def test_backward(mrl, ctx, T, N, heads, key_heads, dk, dv, dtype):
    print("delta backward", T, N, heads, key_heads, dk, dv, dtype, flush=True)
    c = Case(T, N, heads, key_heads, dk, dv, dtype, packed=(T + N + dk) % 2 == 1, dones=(T + dk) % 3 != 0, state=N % 4 != 3)
    got = c.backward(mrl, ctx)
    ctx.synchronize()
    want, terms = c.backward64()
    for name, x, y in zip((*c.NAMES, "state"), got, want):
        per = key_heads if name in ("query", "key") else heads
        near(x, y, per, BACKWARD, UNIT if name == "state" else HALF[dtype], "grad_" + name, terms.get(name))
    again = c.backward(mrl, ctx)
    ctx.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,dk,dv", [(40, 3, 2, 20, 24), (70, 2, 1, 64, 64), (90, 2, 2, 128, 40), (400, 2, 1, 64, 20), (330, 2, 2, 128, 16)])
def test_what_a_cut_hides(mrl, ctx, T, N, heads, dk, dv, dtype):
    """Infinities and NaN in a first state, in keys, values and gates, in output gradients: nothing behind (backwards: ahead of) a cut
    changes, nor do other environments, and steps ahead of a value that is not finite come out as they do without it."""
    def case():
        c = Case(T, N, heads, heads, dk, dv, dtype, dones=True, rate=0.0)
        c.prev[0] = 1.0
        c.dones.view(T, N)[T // 2 - 1, 0] = 1.0
        c.cut = torch.cat((c.prev[None], c.dones[:-1])).cpu() > 0.5
        return c
    clean, bad = case(), case()
    out, last = clean.forward(mrl, ctx)
    grads = clean.backward(mrl, ctx)
    bad.state[0] = float("nan")                   # hidden by the cut ahead of the first step
    at = (T // 2 - 5) * N                          # a step of environment 0 before its second cut
    bad.rows[2].view(-1, heads * dv)[at, 3] = float("inf")
    bad.rows[1][at + N, 1] = float("nan")
    bad.grad_out[at, 0] = float("nan")
    bad.rows[3][at + 2 * N, 0] = float("nan")
    got, got_last = bad.forward(mrl, ctx)
    got_grads = bad.backward(mrl, ctx)
    ctx.synchronize()
    off = 2 * FORWARD
    def by_step(x):
        return x.view(T, N, -1).cpu().double()
    x, y = by_step(got), by_step(out)
    half = HALF[dtype]
    def same(a, b, off):
        assert torch.isfinite(a).all()
        assert ((a - b).abs() <= off * b.abs().max() + 2 * half * b.abs()).all()
    same(x[:, 1:], y[:, 1:], off)                 # other environments
    same(x[T // 2:, 0], y[T // 2:, 0], off)       # behind the cut
    same(x[:T // 2 - 5, 0], y[:T // 2 - 5, 0], off)   # ahead of the first value that is not finite
    assert not torch.isfinite(x[T // 2 - 5, 0]).all()
    same(got_last.cpu().double(), last.cpu().double(), off)
    for name, a, b in zip(clean.NAMES, got_grads, grads):
        a, b = by_step(a), by_step(b)
        same(a[:, 1:], b[:, 1:], 2 * BACKWARD)
        same(a[T // 2:, 0], b[T // 2:, 0], 2 * BACKWARD)
        if name == "gate":
            assert (a[0, 0] == 0).all()           # nothing goes back through a cut
    first = got_grads[5].cpu().double()
    assert (first[0] == 0).all()
    same(first[1:], grads[5].cpu().double()[1:], 2 * BACKWARD)


# ---- calls other than one pass over a rollout with outputs of its own
def step_rows(c, first, last):
    return [x[first * c.N:last * c.N] for x in c.rows]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,key_heads,dk,dv,lengths", [(21, 5, 2, 1, 24, 40, [1] * 21), (200, 3, 1, 1, 128, 128, [1, 2, 3, 4, 5, 70, 16, 99]), (900, 2, 2, 2, 64, 32, [300, 1, 599])])
def test_in_pieces_with_the_state_in_place(mrl, ctx, T, N, heads, key_heads, dk, dv, lengths, dtype):
    """A rollout in pieces, single steps among them, the state updated where it is: what 64 bits give for the whole of it."""
    c = Case(T, N, heads, key_heads, dk, dv, dtype, packed=True, seed=4)
    state, prev, at = c.state.clone(), c.prev, 0
    wide = torch.full((T * N, 2 + heads * dv), 7.0, dtype=c.tt, device="cuda")
    out = wide[:, 1:-1]
    for n in lengths:
        rows, o = step_rows(c, at, at + n), out[at * N:(at + n) * N]
        if n == 1:
            c.layer(mrl).step_gpu(ctx, o, *rows, state, prev_dones=prev)
        else:
            c.layer(mrl).forward_gpu(ctx, o, *rows, n, state_in=state, state_out=state, dones=c.dones[at:at + n], prev_dones=prev)
        at += n
        prev = c.dones[at - 1]
    assert at == T
    ctx.synchronize()
    want, want_last = c.forward64()
    near(out.contiguous(), want, heads, FORWARD, HALF[dtype], "out")
    near(state, want_last, heads, FORWARD, UNIT, "state")
    assert (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,dk,dv", [(1, 70, 2, 16, 20), (50, 3, 2, 64, 24), (700, 2, 1, 40, 64), (600, 1, 1, 128, 128)])
def test_states_and_their_gradients_in_place(mrl, ctx, T, N, heads, dk, dv, dtype):
    c = Case(T, N, heads, heads, dk, dv, dtype, seed=6)
    out, last = c.forward(mrl, ctx)
    grads = c.backward(mrl, ctx)
    state, grad_state = c.state.clone(), c.grad_last.clone()
    again, mine = torch.empty_like(out), [torch.empty_like(g) for g in grads[:5]]
    c.layer(mrl).backward_gpu(ctx, *mine, c.grad_out, *c.rows, T, state_in=state, dones=c.dones, prev_dones=c.prev, grad_state_out=grad_state, grad_state_in=grad_state)
    c.layer(mrl).forward_gpu(ctx, again, *c.rows, T, state_in=state, state_out=state, dones=c.dones, prev_dones=c.prev)
    ctx.synchronize()
    assert torch.equal(again, out) and torch.equal(state, last) and torch.equal(grad_state, grads[5]) and all(torch.equal(a, b) for a, b in zip(mine, grads))


@pytest.mark.parametrize("T,N,dk", [(40, 2, 16), (500, 1, 24)])
def test_gradient_against_differences(mrl, ctx, T, N, dk):
    """Directional derivatives of the rule in 64 bits, taken as differences."""
    c = Case(T, N, 2, 1, dk, 12, "f32", seed=8)
    grads = c.backward(mrl, ctx)
    ctx.synchronize()
    inputs = [*c.rows64(), c.state64()]
    weights, last = c.grad_out.cpu().double(), c.grad_last.cpu().double()

    def loss(at):
        out, end, _, _ = rule64(at[:5], at[5], c.cut, *c.dims)
        return ((out.reshape(T * N, -1) * weights).sum() + (end * last).sum()).item()
    gen = torch.Generator().manual_seed(5)
    size = weights.abs().sum().item() + last.abs().sum().item()
    for which, grad in enumerate(grads):
        grad = grad.cpu().double()
        v = torch.randn(inputs[which].shape, generator=gen, dtype=torch.float64)
        eps = 1e-5
        up, down = list(inputs), list(inputs)
        up[which], down[which] = inputs[which] + eps * v, inputs[which] - eps * v
        want = (loss(up) - loss(down)) / (2 * eps)
        # differences: eps^2 of third derivatives and 2^-52 / eps of the loss's terms; the gradient's own bound for every value
        assert abs((grad * v).sum().item() - want) <= BACKWARD * grad.abs().max().item() * v.abs().sum().item() + 1e-8 * size, c.NAMES[which:which + 1]


def test_gates_and_rates_at_their_ends(mrl, ctx):
    """Gates and rates that are 0 or 1 to the last bit, infinite ones among them, and rows of zeros for keys and queries."""
    for dtype in ("f32", "bf16"):
        c = Case(80, 2, 2, 2, 16, 24, dtype, dones=False, seed=9)
        q, k, v, gate, rate = c.rows
        gate[3], gate[20], gate[41], gate[60] = -float("inf"), float("inf"), -200.0, 200.0
        rate[5], rate[21], rate[43], rate[61] = -float("inf"), float("inf"), -200.0, 200.0
        k[30], q[31], k[77], q[77] = 0, 0, 0, 0
        out, last = c.forward(mrl, ctx)
        grads = c.backward(mrl, ctx)
        ctx.synchronize()
        want, want_last = c.forward64()
        near(out, want, 2, FORWARD, HALF[dtype], "out")
        near(last, want_last, 2, FORWARD, UNIT, "state_out")
        wants, terms = c.backward64()
        for name, x, y in zip((*c.NAMES, "state"), grads, wants):
            near(x, y, 2, BACKWARD, UNIT if name == "state" else HALF[dtype], "grad_" + name, terms.get(name))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_other_streams_and_captured_graphs(mrl, ctx, dtype):
    """Two graphs of one context's calls, each with a workspace of its own, replayed on different streams with eager calls between."""
    cases = [Case(700, 2, 2, 1, 40, 24, dtype, seed=1), Case(65, 20, 1, 1, 128, 64, dtype, seed=2)]
    wants = [(*c.forward(mrl, ctx), *c.backward(mrl, ctx)) for c in cases]
    ctx.synchronize()
    side = torch.cuda.Stream()
    cctx = mrl.DeviceContext("cuda:0", stream=side)
    graphs, outs = [], []
    for c in cases:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append((*c.forward(mrl, cctx), *c.backward(mrl, cctx)))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for o in outs:
            for t in o:
                t.fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = cases[0].forward(mrl, ctx)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager, wants[0]))
        for o, w in zip(outs, wants):
            assert all(torch.equal(x, y) for x, y in zip(o, w))
    del graphs
    cctx.close()


def test_no_steps_and_no_environments(mrl, ctx):
    lib = mrl._lib.lib()
    a, b = torch.randn(48, device="cuda"), torch.zeros(48, device="cuda")
    d = mrl._lib.Delta(0, 0, 3, 1, 1, 4, 4, *(None,) * 5, *(0,) * 5, None, None, a.data_ptr())
    p, none = ctypes.c_void_p(b.data_ptr()), mrl._lib.DeltaGrads()
    assert lib.mrl_delta_forward(ctx.handle, ctypes.byref(d), None, 0, p, None, 0) == 0
    ctx.synchronize()
    assert torch.equal(a, b)
    none.state = b.data_ptr()
    assert lib.mrl_delta_backward(ctx.handle, ctypes.byref(d), None, 0, None, ctypes.byref(none), None, 0) == 0
    ctx.synchronize()
    assert not b.any()
    layer = mrl.GatedDeltaRule(2, 4, 3)
    empty = [torch.empty(0, w, device="cuda") for w in (6, 8, 8, 6, 2, 2)]
    layer.forward_gpu(ctx, *empty, 5)
    layer.backward_gpu(ctx, *empty[1:], *empty, 5)
    ctx.synchronize()


def test_library_refusals(mrl, ctx):
    lib, x, size = mrl._lib.lib(), torch.zeros(1 << 18, device="cuda"), ctypes.c_uint64(0)
    at = x.data_ptr()
    far = at + 4 * (1 << 17)

    def description(**other):
        d = mrl._lib.Delta(0, 10, 3, 2, 1, 4, 4, at, at, at, at, at, 4, 4, 8, 2, 2, None, None, None)
        for name, value in other.items():
            setattr(d, name, value)
        return d
    for bad, text in ((dict(dtype=2), b"element type"), (dict(T=-1), b"negative"), (dict(T=1 << 30), b"2^30"), (dict(N=1 << 21), b"2^22"), (dict(heads=3, key_heads=2), b"heads"),
                      (dict(key_dim=129), b"dim"), (dict(value_dim=0), b"dim"), (dict(key=None), b"NULL"), (dict(query_ld=3), b"stride"), (dict(rate_ld=1), b"stride")):
        d = description(**bad)
        assert lib.mrl_delta_forward(ctx.handle, ctypes.byref(d), far, 8, None, None, 0) == -1 and text in lib.mrl_last_error(), (bad, lib.mrl_last_error())
    assert lib.mrl_delta_forward(ctx.handle, ctypes.byref(description()), None, 8, None, None, 0) == -1 and b"NULL" in lib.mrl_last_error()
    assert lib.mrl_delta_forward(ctx.handle, ctypes.byref(description()), far, 7, None, None, 0) == -1 and b"stride" in lib.mrl_last_error()
    grads = mrl._lib.DeltaGrads(far, far + 4096, far + 8192, far + 12288, far + 16384, 4, 4, 8, 2, 2, None)
    d = description(T=2000, N=1)
    for backward in (0, 1):
        assert lib.mrl_delta_workspace(ctx.handle, ctypes.byref(d), backward, ctypes.byref(size)) == 0 and 0 < size.value
        for ws, n, text in ((None, 0, b"workspace"), (far + 32768 * 4, size.value - 1, b"workspace"), (far + 32768 * 4 + 4, size.value, b"aligned")):
            if backward:
                rc = lib.mrl_delta_backward(ctx.handle, ctypes.byref(d), at, 8, None, ctypes.byref(grads), ws, n)
            else:
                rc = lib.mrl_delta_forward(ctx.handle, ctypes.byref(d), far, 8, None, ws, n)
            assert rc == -1 and text in lib.mrl_last_error(), lib.mrl_last_error()
    ctx.synchronize()
    assert not x.any()


def test_outputs_on_inputs_are_refused(mrl, ctx):
    """Before anything is launched: the buffers stay as they are."""
    c = Case(40, 3, 2, 2, 8, 8, "f32", packed=True)
    wide = c.rows[0]._base if c.rows[0]._base is not None else c.rows[0]
    before = wide.clone()
    out = torch.zeros(120, 16, device="cuda")
    grads = [torch.zeros(120, w, device="cuda") for w in c.widths]
    flat = torch.zeros(4, 3 * 2 * 64, device="cuda")

    def forward(**other):
        c.layer(mrl).forward_gpu(ctx, **{**dict(zip(c.NAMES, c.rows)), **dict(output=out, steps=40, state_in=flat[0], state_out=flat[1], dones=c.dones, prev_dones=c.prev), **other})

    def backward(**other):
        c.layer(mrl).backward_gpu(ctx, **{**dict(zip(c.NAMES, c.rows)), **dict(zip(("grad_" + n for n in c.NAMES), grads)),
                                          **dict(grad_output=out, steps=40, state_in=flat[0], dones=c.dones, prev_dones=c.prev, grad_state_out=flat[2], grad_state_in=flat[3]), **other})
    for bad in (dict(output=c.rows[2]), dict(output=wide[:, 8:24]), dict(output=wide[:, 36:52]), dict(state_out=flat.view(-1)[5:5 + 384]), dict(dones=out.view(-1)[:120]),
                dict(state_out=out.view(-1)[:384]), dict(prev_dones=flat[1][:3])):
        with pytest.raises(mrl.MrlError, match="overlap"):
            forward(**bad)
    for bad in (dict(grad_query=c.rows[0]), dict(grad_query=grads[1]), dict(grad_value=out), dict(grad_gate=grads[4]), dict(grad_state_in=flat[0]),
                dict(grad_state_out=flat.view(-1)[3 * 384 - 1:4 * 384 - 1]), dict(grad_rate=wide[:, 40:42])):
        with pytest.raises(mrl.MrlError, match="overlap"):
            backward(**bad)
    ctx.synchronize()
    assert torch.equal(wide, before) and not out.any() and not flat.any() and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_far_apart(mrl, ctx, dtype):
    """Rows whose last element is past 2^31 elements and 2^32 bytes from the first."""
    ld = 1 << 25
    c = Case(70, 2, 1, 1, 20, 12, dtype, seed=3)
    room = torch.empty(140 * ld, dtype=c.tt, device="cuda")
    wide = room.view(140, ld)
    widths = [*c.widths, 12]
    places = [(1 << 24) + 100 * i + 1 for i in range(12)]
    near_rows, near_out, near_grads = c.rows, torch.empty(140, 12, dtype=c.tt, device="cuda"), [torch.empty(140, w, dtype=c.tt, device="cuda") for w in c.widths]
    far = [wide[:, at:at + w] for at, w in zip(places, widths + list(c.widths) + [12])]
    for f, r in zip(far, near_rows):
        f.copy_(r)
    far[11].copy_(c.grad_out)
    layer = c.layer(mrl)
    for rows, out, grads, grad in ((near_rows, near_out, near_grads, c.grad_out), (far[:5], far[5], far[6:11], far[11])):
        layer.forward_gpu(ctx, out, *rows, 70, state_in=c.state, dones=c.dones, prev_dones=c.prev)
        layer.backward_gpu(ctx, *grads, grad, *rows, 70, state_in=c.state, dones=c.dones, prev_dones=c.prev)
    step = torch.empty(2, 12, dtype=c.tt, device="cuda"), far[5][138:]
    for rows, out in ((near_rows, step[0]), (far[:5], step[1])):
        layer.step_gpu(ctx, out, *[r[138:] for r in rows], c.state.clone())
    ctx.synchronize()
    assert torch.equal(step[0], step[1]) and all(torch.equal(a, b) for a, b in zip(near_grads, far[6:11]))
    assert torch.equal(near_out[:138], far[5][:138])


# ---- parts with and without cuts
def parts_of(T, N, heads, dk, dv):
    """steps of a part of a long rollout, and the number of parts (parts_of in delta.hpp)"""
    block = 32 if dk > 32 else 64
    blocks = -(-T // block)
    groups = N * heads * ((-(-dv // 16) + 7) // 8)
    want = min(blocks, 2 * torch.cuda.get_device_properties(0).multi_processor_count // groups, int((20.0 * blocks) ** 0.5), 1024)
    per = -(-blocks // want)
    return per * block, -(-blocks // per)


# by part: whether a cut is ahead of one of its steps (the first, the last, or both)
PATTERNS = {"every second": ".x" * 16, "and the others": "x." * 16, "two without around one": "..x" * 11, "two with around one": "xx." * 11, "once": ".........x......", "none": "." * 16}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pattern,where", [(p, w) for p in PATTERNS for w in ("first", "last", "both") if p != "none" or w == "first"])
@pytest.mark.parametrize("T,N,heads,key_heads,dk,dv", [(700, 1, 1, 1, 12, 20), (1020, 2, 2, 1, 24, 40), (630, 1, 2, 2, 60, 33), (610, 2, 1, 1, 128, 24)])
def test_parts_with_and_without_cuts(mrl, ctx, T, N, heads, key_heads, dk, dv, pattern, where, dtype):
    """What goes from part to part, where some of them have cuts, against 64 bits: outputs, last states and gradients."""
    steps, count = parts_of(T, N, heads, dk, dv)
    assert count >= 8
    print("delta parts", T, N, heads, key_heads, dk, dv, pattern, where, dtype, steps, count, flush=True)
    c = Case(T, N, heads, key_heads, dk, dv, dtype, rate=0.0, seed=12)
    # memories of some tens of steps, as the bounds take them, in every head: what a part leaves reaches the parts behind it
    c.rows[3].copy_(torch.randn(c.rows[3].shape, generator=torch.Generator().manual_seed(T)) + 4)
    flags = torch.zeros(T + 1, N)
    for part in range(count):
        begin, end = part * steps, min(T, (part + 1) * steps)
        if PATTERNS[pattern][part % len(PATTERNS[pattern])] == "x":
            for at in {"first": [begin], "last": [end - 1], "both": [begin, end - 1]}[where]:
                flags[at] = 1.0
    c.prev, c.dones, c.cut = flags[0].cuda(), flags[1:].contiguous().cuda(), flags[:-1] > 0.5
    out, last = c.forward(mrl, ctx)
    got = c.backward(mrl, ctx)
    ctx.synchronize()
    want, want_last = c.forward64()
    near(out, want, heads, FORWARD, HALF[dtype], "out")
    near(last, want_last, heads, FORWARD, UNIT, "state_out")
    wants, terms = c.backward64()
    for name, x, y in zip((*c.NAMES, "state"), got, wants):
        near(x, y, key_heads if name in ("query", "key") else heads, BACKWARD, UNIT if name == "state" else HALF[dtype], "grad_" + name, terms.get(name))
    for _ in range(3):   # nor does it depend on which wavefront is ahead
        again, again_last = c.forward(mrl, ctx)
        more = c.backward(mrl, ctx)
        ctx.synchronize()
        assert torch.equal(out, again) and torch.equal(last, again_last) and all(torch.equal(x, y) for x, y in zip(got, more))


# ---- the ends of the range
def by_episode(c, x):
    """the parts of [T, N, ...] that cuts separate, by environment"""
    x = x.reshape(c.T, c.N, *x.shape[1:])
    for n in range(c.N):
        starts = [0, *[t for t in range(1, c.T) if c.cut[t, n]], c.T]
        for first, last in zip(starts, starts[1:]):
            yield x[first:last, n]


def sums_of_terms(c):
    """What roundings in the gradients of gate and rate are of the size of.  grad_gate = (1 - a) sum_ij S'[i][j] dS'[i][j] is a sum of dk dv terms,
    grad_rate = (1 - b) sum_j U[j] dX[j] of dv, and either may be far smaller than they are (1280 terms that cancel to a 3000th of their 2-norm
    in the first step of 600, the only one that meets the first state).  A term is off by its factors' bounds, one term independently of another, so the sum is off
    by those times the terms' 2-norm.  The terms are the gradients of a gate for every element of the state, and a rate for every column."""
    heads, key_heads, dk, dv = c.dims
    T, N = c.T, c.N
    q, k, v, gate, rate = c.rows64()
    q, k = (x.reshape(T, N, key_heads, dk) for x in (q, k))
    q, k = ((x / (x.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(heads // key_heads, 2) for x in (q, k))
    v = v.reshape(T, N, heads, dv)
    a = torch.sigmoid(gate).reshape(T, N, heads, 1, 1).expand(T, N, heads, dk, dv).clone().requires_grad_()
    b = torch.sigmoid(rate).reshape(T, N, heads, 1, 1).expand(T, N, heads, 1, dv).clone().requires_grad_()
    state, loss, weights = c.state64(), 0.0, c.grad_out.cpu().double().reshape(T, N, heads, dv) / dk ** 0.5
    for t in range(T):
        state = torch.where(c.cut[t].view(N, 1, 1, 1), torch.zeros_like(state), a[t] * state)
        state = state + k[t].unsqueeze(3) * (b[t] * (v[t].unsqueeze(2) - k[t].unsqueeze(2) @ state))
        loss = loss + ((q[t].unsqueeze(2) @ state).squeeze(2) * weights[t]).sum()
    of_a, of_b = torch.autograd.grad(loss + (state * c.grad_last.cpu().double()).sum(), [a, b])
    return {name: (p * (1 - p) * g).detach().norm(dim=(3, 4)).reshape(T * N, heads) for name, p, g in (("gate", a, of_a), ("rate", b, of_b))}


# (steps: by the state's own pass, within a tile, over tiles, in parts)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,N,heads,key_heads,dk,dv", [(1, 3, 2, 2, 64, 64), (4, 2, 2, 1, 40, 24), (3, 1, 1, 1, 128, 100), (30, 2, 2, 1, 24, 40), (70, 2, 1, 1, 128, 64), (45, 2, 2, 2, 9, 5), (600, 1, 1, 1, 64, 20)])
@pytest.mark.parametrize("keys,queries,states", [(1e12, 1.0, 1e29), (1.0, 5e17, 1.0), (1e25, 1e25, 1.0), (1e19, 1e-3, 1e30), (1e-12, 1e-12, 1e33), (3e36, 3e36, 1e-20), (1.0, 1.0, 1e35)])
def test_sizes_of_keys_queries_and_states(mrl, ctx, T, N, heads, key_heads, dk, dv, keys, queries, states, dtype):
    """A key's and a query's length go out of the results, so that their products with a state are of the state's size; and what large ones make
    of the steps ahead of a cut does not reach those behind it.  Against 64 bits, episode by episode."""
    print("delta range", T, N, heads, key_heads, dk, dv, keys, queries, states, dtype, flush=True)
    c = Case(T, N, heads, key_heads, dk, dv, dtype, rate=0.0, seed=14)
    if T > 4:   # in the middle of a tile
        c.dones[T // 2 - 1] = 1.0
        c.cut = torch.cat((c.prev[None], c.dones[:-1])).cpu() > 0.5
    c.rows[0].mul_(queries)
    c.rows[1].mul_(keys)
    c.state.mul_(states)
    out, last = c.forward(mrl, ctx)
    got = c.backward(mrl, ctx)
    ctx.synchronize()
    want, want_last = c.forward64()
    near(last, want_last, heads, FORWARD, UNIT, "state_out")
    for x, y in zip(by_episode(c, out.cpu().double()), by_episode(c, want)):
        near(x, y, heads, FORWARD, HALF[dtype], "out")
    wants, terms = c.backward64()
    terms.update(sums_of_terms(c))
    for name, x, y in zip((*c.NAMES, "state"), got, wants):
        if name == "state":
            near(x, y, heads, BACKWARD, UNIT, "grad_state")
            continue
        size = torch.maximum(terms.get(name, y).detach().abs(), y.detach().abs())
        for a, b, s in zip(by_episode(c, x.cpu().double()), by_episode(c, y), by_episode(c, size)):
            near(a, b, key_heads if name in ("query", "key") else heads, BACKWARD, HALF[dtype], "grad_" + name, s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_cut_within_a_tile_of_large_products(mrl, ctx, dtype):
    """A state, keys, values and output gradients whose products with each other pass fp32's end, in the steps ahead of a cut: those behind it
    come out as they do without them."""
    T, N, heads, dk, dv = 90, 2, 2, 24, 20

    def case():
        c = Case(T, N, heads, heads, dk, dv, dtype, rate=0.0, seed=15)
        c.dones[40] = 1.0
        c.cut = torch.cat((c.prev[None], c.dones[:-1])).cpu() > 0.5
        return c
    clean, bad = case(), case()
    rows = slice(36 * N, 41 * N)
    bad.state.mul_(1e28)
    for which, by in ((0, 1e15), (1, 1e14), (2, 1e25)):
        bad.rows[which][rows] *= by
    bad.grad_out[rows] *= 1e27
    results = [(*c.forward(mrl, ctx), *c.backward(mrl, ctx)) for c in (clean, bad)]
    ctx.synchronize()
    for x, y in zip(results[1][:1] + results[1][2:7], results[0][:1] + results[0][2:7]):
        x, y = x.cpu().double()[41 * N:], y.cpu().double()[41 * N:]
        assert torch.isfinite(x).all() and ((x - y).abs() <= 2 * BACKWARD * y.abs().max() + 2 * HALF[dtype] * y.abs()).all()
    assert (results[1][1].cpu().double() - results[0][1].cpu().double()).abs().max() <= 2 * FORWARD * results[0][1].abs().max().item()
