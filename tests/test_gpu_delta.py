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
