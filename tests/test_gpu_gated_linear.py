"""GatedLinear against its formulas and their gradients in 64 bits."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": UNIT, "bf16": 2.0 ** -8}
# Roundings of a sum of n products at its full size: six additions to the sum for every 32 products (one in bf16), those of up to 64 partial sums
# and of the bias, and 2 units of each product, for the pieces left out.
ROUNDINGS = lambda n: (6 * n / 32 + 72) * UNIT   # noqa: E731
ACTIVATIONS = ("sigmoid", "silu", "gelu", "tanh")


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


def act64(act, g):
    s = torch.sigmoid(g)
    return {"sigmoid": s, "silu": g * s, "gelu": 0.5 * g * (1 + torch.erf(g / math.sqrt(2))), "tanh": torch.tanh(g)}[act]


class Case:
    def __init__(self, M, K, N, act, dtype, seed=0, wide=False):
        gen = torch.Generator().manual_seed(seed + 7 * M + 5 * K + N)
        self.M, self.K, self.N, self.act, self.dtype, self.tt = M, K, N, act, dtype, TYPES[dtype]
        x = torch.randn(M, K, generator=gen).to(self.tt)
        params = torch.cat((torch.randn(K * 2 * N, generator=gen) / math.sqrt(K), torch.randn(2 * N, generator=gen) * 0.2)).to(self.tt)
        grad = torch.randn(M, N, generator=gen).to(self.tt)
        if wide:     # rows farther apart than they are long, at odd places
            room = torch.zeros(M, K + N + 5, dtype=self.tt)
            room[:, 1:1 + K], room[:, K + 3:K + 3 + N] = x, grad
            room = room.cuda()
            self.x, self.grad = room[:, 1:1 + K], room[:, K + 3:K + 3 + N]
        else:
            self.x, self.grad = x.cuda(), grad.cuda()
        self.params = params.cuda()

    def parts64(self):
        x, p, grad = self.x.cpu().double(), self.params.cpu().double(), self.grad.cpu().double()
        K, N = self.K, self.N
        w = p[:K * 2 * N].view(K, 2 * N)
        pre = x @ w + p[K * 2 * N:]
        off = ROUNDINGS(K) * (x.abs() @ w.abs() + p[K * 2 * N:].abs())
        return x, w, grad, pre, off

    def forward64(self):
        """outputs and what they may be off by: activations' slopes are at most 1.13; their values take some ten roundings"""
        x, w, grad, pre, off = self.parts64()
        g, u, og, ou = pre[:, :self.N], pre[:, self.N:], off[:, :self.N], off[:, self.N:]
        a = act64(self.act, g)
        return a * u, 1.13 * og * (u.abs() + ou) + (a.abs() + 16 * UNIT * (1 + g.abs())) * ou + 16 * UNIT * (a.abs() + UNIT) * u.abs() + HALF[self.dtype] * (a * u).abs() + 1e-37

    def backward64(self):
        """(grad_x, what it may be off by), (grads, ...): the slopes' slopes are at most 1; a slope takes some twenty roundings of terms up to
        1 + |g|.  In bf16 [dgate | dup] is rounded for grad_x, half a step, and taken as two pieces, 2^-17, for the parameters."""
        x, w, grad, pre, off = self.parts64()
        N = self.N
        g = pre[:, :N].clone().requires_grad_()
        a = act64(self.act, g)
        slope, = torch.autograd.grad(a.sum(), g)
        g, a = g.detach(), a.detach()
        u, og, ou = pre[:, N:], off[:, :N], off[:, N:]
        d = torch.cat((grad * u * slope, grad * a), 1)
        few = 24 * UNIT * (1 + g.abs().clamp(max=8))
        od = torch.cat((grad.abs() * (ou * (slope.abs() + few) + u.abs() * (og + few)), grad.abs() * (1.13 * og + few)), 1)
        piece, pieces = (2.0 ** -8, 2.0 ** -17) if self.dtype == "bf16" else (0.0, 0.0)
        gx, ox = d @ w.T, (od + (piece + ROUNDINGS(2 * N)) * d.abs()) @ w.abs().T
        gw, ow = x.T @ d, x.abs().T @ (od + (pieces + ROUNDINGS(self.M)) * d.abs())
        gb, ob = d.sum(0), (od + ROUNDINGS(32 * self.M) * d.abs()).sum(0)
        return (gx, ox + HALF[self.dtype] * gx.abs() + 1e-37), (torch.cat((gw.reshape(-1), gb)), torch.cat((ow.reshape(-1), ob)) + 1e-37)

    def layer(self, mrl):
        return mrl.GatedLinear(self.K, self.N, self.act)

    def forward(self, mrl, ctx):
        out = torch.full((self.M, self.N), 7.0, dtype=self.tt, device="cuda")
        self.layer(mrl).forward_gpu(ctx, out, self.x, self.params)
        return out

    def backward(self, mrl, ctx, grad_x=True):
        gx = torch.full((self.M, self.K), 7.0, dtype=self.tt, device="cuda") if grad_x else None
        grads = torch.full((2 * self.N * (self.K + 1),), 7.0, device="cuda")
        self.layer(mrl).backward_gpu(ctx, gx, grads, self.grad, self.x, self.params)
        return gx, grads


def near(got, want, off, what):
    beyond = (got.cpu().double().reshape(want.shape) - want).abs() - off
    assert beyond.max().item() <= 0, "%s: %g beyond its bound at %d of %s" % (what, beyond.max().item(), beyond.argmax().item(), list(want.shape))


# rows below, at and one past a fragment, a tile and what goes straight to registers; odd dims, dims of one, columns past a tile
SHAPES = [(1, 1, 1), (1, 256, 1024), (16, 64, 48), (17, 33, 31), (64, 100, 20), (65, 32, 16), (66, 7, 5), (127, 96, 130), (128, 64, 128), (129, 65, 129), (300, 256, 7),
          (257, 40, 300), (1000, 128, 64), (513, 520, 272), (2050, 72, 36)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_forward_and_backward(mrl, ctx, M, K, N, dtype):
    act = ACTIVATIONS[(M + K + N) % 4]
    print("gated linear", M, K, N, act, dtype, flush=True)
    c = Case(M, K, N, act, dtype, wide=M % 2 == 1)
    out = c.forward(mrl, ctx)
    ctx.synchronize()
    near(out, *c.forward64(), "out")
    gx, grads = c.backward(mrl, ctx)
    ctx.synchronize()
    for got, (want, off), what in zip((gx, grads), c.backward64(), ("grad_x", "grads")):
        near(got, want, off, what)
    again = c.backward(mrl, ctx)
    _, alone = c.backward(mrl, ctx, grad_x=False)
    ctx.synchronize()
    assert torch.equal(gx, again[0]) and torch.equal(grads, again[1]) and torch.equal(grads, alone)


# on both sides of what goes straight to registers: long products, wide outputs, 256 rows and one more
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 2050, 17), (65, 513, 40), (64, 512, 2064), (127, 1100, 640), (128, 520, 272), (129, 530, 700), (256, 40, 64), (257, 40, 64), (16, 3, 4100), (32, 1040, 4110), (33, 1040, 4110)])
def test_few_rows_and_tiles(mrl, ctx, M, K, N, dtype):
    print("gated linear", M, K, N, dtype, flush=True)
    c = Case(M, K, N, "silu", dtype, wide=M % 2 == 1)
    out = c.forward(mrl, ctx)
    ctx.synchronize()
    near(out, *c.forward64(), "out")


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("M", [30, 200])
def test_activations(mrl, ctx, act, M):
    c = Case(M, 48, 40, act, "f32", seed=3)
    c.params[:48 * 80] *= 6      # gates out to where the activations are flat
    out = c.forward(mrl, ctx)
    gx, grads = c.backward(mrl, ctx)
    ctx.synchronize()
    near(out, *c.forward64(), "out")
    for got, (want, off), what in zip((gx, grads), c.backward64(), ("grad_x", "grads")):
        near(got, want, off, what)


def test_gradient_against_differences(mrl, ctx):
    """a step h along a direction changes the weighted outputs by h times the gradient along it, to h^2 and the outputs' roundings"""
    c = Case(70, 40, 24, "silu", "f32", seed=5)
    gx, grads = c.backward(mrl, ctx)
    gen = torch.Generator().manual_seed(1)
    h = 2.0 ** -6
    weight = c.grad.double()
    for name, grad in (("x", gx), ("params", grads)):
        direction = torch.randn(getattr(c, name).shape, generator=gen).cuda()
        here = getattr(c, name)
        sums = []
        for sign in (1, -1):
            setattr(c, name, here + sign * h * direction)
            sums.append((c.forward(mrl, ctx).double() * weight).sum())
        setattr(c, name, here)
        want = (grad.double() * direction.double()).sum().item()
        got = ((sums[0] - sums[1]) / (2 * h)).item()
        # third derivatives are of the order of the sum of |weight| times cubes of the directions' products, here below 2^8 of the gradient's norm
        norm = (grad.double().norm() * direction.double().norm()).item()
        assert abs(got - want) <= 2.0 ** 8 * h * h / 6 * norm / math.sqrt(direction.numel()) + 1e-3 * norm / math.sqrt(direction.numel())


def test_empty_and_refused(mrl, ctx):
    layer = mrl.GatedLinear(8, 4)
    x, out, params, grads = torch.zeros(0, 8, device="cuda"), torch.zeros(0, 4, device="cuda"), torch.zeros(layer.PARAM_SIZE, device="cuda"), torch.ones(layer.PARAM_SIZE, device="cuda")
    layer.forward_gpu(ctx, out, x, params)
    layer.backward_gpu(ctx, None, grads, out, x, params)
    ctx.synchronize()
    assert (grads == 0).all()
    x, out = torch.zeros(100, 8, device="cuda"), torch.zeros(100, 4, device="cuda")
    with pytest.raises(mrl.MrlError, match="overlap"):
        layer.forward_gpu(ctx, x[:, :4], x, params)
    with pytest.raises(mrl.MrlError, match="overlap"):
        layer.backward_gpu(ctx, x, grads, out, x, params)
    with pytest.raises(mrl.MrlError, match="overlap"):
        layer.backward_gpu(ctx, None, params, out, x, params)
    call, ptr = mrl._lib.call, lambda t: t.data_ptr()   # noqa: E731
    for args, text in (((0, 0, 300, 8, 4, ptr(x), 8, ptr(params), ptr(out), 4, None, 0), "workspace"), ((0, 0, 100, 8, 4, ptr(x), 7, ptr(params), ptr(out), 4, None, 0), "stride"),
                       ((0, 9, 100, 8, 4, ptr(x), 8, ptr(params), ptr(out), 4, None, 0), "activation"), ((7, 0, 100, 8, 4, ptr(x), 8, ptr(params), ptr(out), 4, None, 0), "type"),
                       ((0, 0, 100, 0, 4, ptr(x), 8, ptr(params), ptr(out), 4, None, 0), "dims"), ((0, 0, -1, 8, 4, ptr(x), 8, ptr(params), ptr(out), 4, None, 0), "rows"),
                       ((0, 0, 100, 8, 4, None, 8, ptr(params), ptr(out), 4, None, 0), "NULL")):
        with pytest.raises(mrl.MrlError, match=text):
            call("mrl_gated_linear_forward", ctx.handle, *args)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_other_streams_and_captured_graphs(mrl, ctx, dtype):
    """Two graphs of one context's calls, each with a workspace of its own, replayed on different streams with eager calls between."""
    cases = [Case(1500, 72, 40, "gelu", dtype, seed=1), Case(20, 33, 65, "silu", dtype, seed=2)]
    wants = [(c.forward(mrl, ctx), *c.backward(mrl, ctx)) for c in cases]
    ctx.synchronize()
    side = torch.cuda.Stream()
    cctx = mrl.DeviceContext("cuda:0", stream=side)
    graphs, outs = [], []
    for c in cases:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append((c.forward(mrl, cctx), *c.backward(mrl, cctx)))
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
        assert torch.equal(eager, wants[0][0])
        for o, w in zip(outs, wants):
            assert all(torch.equal(x, y) for x, y in zip(o, w))
    del graphs
    cctx.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M", [40, 300])
def test_rows_that_are_not_finite(mrl, ctx, M, dtype):
    """An infinity or NaN in a row of the input reaches that row of the outputs and of grad_input, and no other."""
    c = Case(M, 70, 50, "silu", dtype, seed=4)
    out, (gx, _) = c.forward(mrl, ctx), c.backward(mrl, ctx)
    c.x[17, 3], c.x[M - 1, 69], c.grad[21, 5] = float("nan"), float("inf"), float("inf")
    bad, (bad_x, bad_grads) = c.forward(mrl, ctx), c.backward(mrl, ctx)
    ctx.synchronize()
    rows = torch.ones(M, dtype=torch.bool)
    rows[[17, M - 1]] = False
    assert torch.equal(bad[rows], out[rows]) and torch.isnan(bad[17]).all() and not torch.isfinite(bad[M - 1]).all()
    rows[21] = False
    assert torch.equal(bad_x[rows], gx[rows]) and not torch.isfinite(bad_x[21]).any() and torch.isnan(bad_x[17]).all()
    assert torch.isnan(bad_grads.view(-1)[:70 * 100].view(70, 100)[3]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M", [140, 300])
def test_rows_far_apart(mrl, ctx, M, dtype):
    """Rows whose last element is past 2^31 elements and 2^32 bytes from the first."""
    ld = 1 << 24
    c = Case(M, 96, 40, "silu", dtype, seed=9)
    wide = torch.empty(M * ld, dtype=c.tt, device="cuda").view(M, ld)
    x, grad, out, gx = (wide[:, at:at + w] for at, w in ((1 << 23, 96), ((1 << 23) + 104, 40), ((1 << 23) + 200, 40), (ld - 96, 96)))
    x.copy_(c.x)
    grad.copy_(c.grad)
    want, (want_x, want_grads) = c.forward(mrl, ctx), c.backward(mrl, ctx)
    grads = torch.empty_like(want_grads)
    c.layer(mrl).forward_gpu(ctx, out, x, c.params)
    c.layer(mrl).backward_gpu(ctx, gx, grads, grad, x, c.params)
    ctx.synchronize()
    assert torch.equal(out, want) and torch.equal(gx, want_x) and torch.equal(grads, want_grads)


@pytest.mark.parametrize("M", [40, 16383, 16384])
def test_pieces_of_the_parameters_gradient(mrl, ctx, M):
    """In bf16: below 2^14 rows the gradient's terms have 22 bits, from there on 16."""
    c = Case(M, 24, 20, "silu", "bf16", seed=11)
    _, grads = c.backward(mrl, ctx)
    ctx.synchronize()
    _, (want, off) = c.backward64()
    near(grads, want, off, "grads")
    # A sum's terms are off independently of each other, each by at most 2^-22 or 2^-16 of itself and by the roundings of the activation's slope, some 24
    # units; a running sum by half a unit of itself, 6 times for every 32 rows: in the 2-norm over all sums their root squares add.
    rows = math.sqrt(6 * M / 32)
    bound = (2.0 ** -22 + 24 * UNIT + rows * UNIT) if M < 1 << 14 else 2.0 ** -16 + 24 * UNIT + rows * UNIT
    assert (grads.cpu().double() - want).norm() <= bound * want.norm()


@pytest.mark.parametrize("M,K,N", [(40, 24, 20), (300, 96, 130), (2050, 72, 36), (513, 520, 272), (4200, 1030, 520)])
def test_grad_input_in_bf16_is_rounded_once(mrl, ctx, M, K, N):
    """Its terms have 16 bits: beside storing's half step of the value there is 2^-17 of each term, which a sum that cancels shows, and no 2^-8."""
    c = Case(M, K, N, "silu", "bf16", seed=12)
    gx, _ = c.backward(mrl, ctx)
    ctx.synchronize()
    x, w, grad, pre, off = c.parts64()
    g, u = pre[:, :N], pre[:, N:]
    s = torch.sigmoid(g)
    slope = s * (1 + g * (1 - s))
    d = torch.cat((grad * u * slope, grad * g * s), 1)
    few = 24 * UNIT * (1 + g.abs().clamp(max=8))
    og, ou = off[:, :N], off[:, N:]
    od = torch.cat((grad.abs() * (ou * (slope.abs() + few) + u.abs() * (og + few)), grad.abs() * (1.13 * og + few)), 1)
    want = d @ w.T
    near(gx, want, (od + (2.0 ** -17 + ROUNDINGS(2 * N)) * d.abs()) @ w.abs().T + HALF["bf16"] * want.abs() + 1e-37, "grad_x")


@pytest.mark.parametrize("M", [300, 16383, 16384, 40000])
def test_the_parameters_gradient_has_the_terms_of_fp32(mrl, ctx, M):
    """Whatever the number of rows.  All but eight rows of the input are zeros, so that the matrix' gradient has eight terms a sum and hardly any
    roundings but those of the terms: 2^-22 for the pieces, 24 units for the activation's value and slope, 8 for the sums."""
    c = Case(M, 24, 20, "silu", "bf16", seed=13)
    some = torch.randperm(M, generator=torch.Generator().manual_seed(3))[:8]
    kept = torch.zeros(M, 1, dtype=c.tt)
    kept[some] = 1
    c.x.mul_(kept.cuda())
    _, grads = c.backward(mrl, ctx)
    ctx.synchronize()
    _, (want, _) = c.backward64()
    got, want = grads.cpu().double()[:24 * 40], want[:24 * 40]
    assert (got - want).norm() <= (2.0 ** -22 + 32 * UNIT) * want.norm()


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M", [3, 300])
def test_gates_far_below_zero(mrl, ctx, M, dtype, act):
    """sigmoid(g) and g sigmoid(g) vanish for the largest gates, in value and slope.  16 units of a value, and the steps of 2^-149 in which
    fp32 goes below 2^-126, up to 110 times.  bf16 goes in steps of 2^-133 there: storing costs half of one, and so do a value's three pieces."""
    gates = torch.tensor([-3e38, -1e38, -1e30, -1e10, -1000.0, -200.0, -110.0, -100.0, -90.0, -88.0, -87.0, -86.0, -30.0, -1.0, 50.0, 1e4])
    N = len(gates)
    params = torch.cat((gates, torch.full((N,), 2.0), torch.zeros(2 * N))).to(TYPES[dtype])
    x, grad = (torch.ones(M, w, dtype=TYPES[dtype], device="cuda") for w in (1, N))
    out, gx, grads = torch.full_like(grad, 7.0), torch.full_like(x, 7.0), torch.full((4 * N,), 7.0, device="cuda")
    layer = mrl.GatedLinear(1, N, act)
    layer.forward_gpu(ctx, out, x, params.cuda())
    layer.backward_gpu(ctx, gx, grads, grad, x, params.cuda())
    ctx.synchronize()
    g = params[:N].double().requires_grad_()
    value = act64(act, g)
    slope, = torch.autograd.grad(value.sum(), g)
    value = value.detach()
    off = 16 * UNIT * value.abs() + 110 * 2.0 ** -149
    assert ((out.cpu().double() - 2 * value).abs() <= 2 * off + HALF[dtype] * 2 * value.abs() + (2.0 ** -134 if dtype == "bf16" else 0.0)).all()
    got = grads.cpu().double().view(2, 2, N)    # matrix and biases, of gate and up
    off = 110 * 2.0 ** -149 + 2.0 ** -134
    steps = (16 + 6 * M) * UNIT                 # a sum over M rows of one value
    assert ((got[:, 0] - 2 * M * slope).abs() <= 2 * M * (steps * slope.abs() + 16 * UNIT * value.abs() + off)).all()
    assert ((got[:, 1] - M * value).abs() <= M * (steps * value.abs() + off)).all()


def kinds(x):
    """0 where finite, 1 and -1 infinities, 2 NaN"""
    return torch.where(torch.isnan(x), 2.0, torch.where(torch.isinf(x), torch.sign(x), torch.zeros_like(x)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("M", [5, 40, 300, 1100])
def test_infinities_are_what_the_formulas_make_of_them(mrl, ctx, M, act, dtype):
    """Whatever the number of rows: infinities in the input, in the matrix' gate and up columns, and in the gradient of the output; and an input
    that is finite and rounds past bf16's largest value."""
    K, N = 70, 50
    for where in ("input", "gate", "up", "grad", "largest"):
        c = Case(M, K, N, act, dtype, seed=21)
        if where == "input":
            c.x[2, 3], c.x[4, 69] = float("inf"), -float("inf")
        elif where == "largest":
            c.x[2, 3] = torch.finfo(c.tt).max        # 2^128, times weights and gradients with which all stays far from overflowing
            c.params[3 * 2 * N:4 * 2 * N] = 2.0 ** -120
            c.grad[2] *= 2.0 ** -20
        elif where == "grad":
            c.grad[1, 7], c.grad[3, 49] = float("inf"), -float("inf")
        else:
            c.params[5 * 2 * N + (0 if where == "gate" else N) + 11] = float("inf")
        out = c.forward(mrl, ctx)
        gx, grads = c.backward(mrl, ctx)
        ctx.synchronize()
        x, p, grad = c.x.cpu().double(), c.params.cpu().double(), c.grad.cpu().double()
        w = p[:K * 2 * N].view(K, 2 * N)
        pre = x @ w + p[K * 2 * N:]
        g = pre[:, :N].clone().requires_grad_()
        a = act64(act, g)
        slope, = torch.autograd.grad(a.sum(), g)
        d = torch.cat((grad * pre[:, N:] * slope, grad * a.detach()), 1)
        want_grads = torch.cat(((x.T @ d).reshape(-1), d.sum(0)))
        for got, want, what in ((out, a.detach() * pre[:, N:], "out"), (gx, d @ w.T, "grad_x"), (grads, want_grads, "grads")):
            want = kinds(want.to(got.dtype).double())
            assert torch.equal(kinds(got.cpu().double()).reshape(want.shape), want), (where, what)


def test_more_operands_than_a_launch_has_threads(mrl, ctx):
    """2^34 values of x, which the gradient lays out twice, in more than 2^32 threads.  Only some rows are not zeros."""
    M, K, N = (1 << 25) + 5, 513, 3
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GiB of device memory")
    some = [0, 12345, (1 << 24) + 3, M - 1]
    c = Case(len(some), K, N, "silu", "bf16", seed=17)
    x, grad = torch.zeros(M, K, dtype=c.tt, device="cuda"), torch.zeros(M, N, dtype=c.tt, device="cuda")
    x[some], grad[some] = c.x, c.grad
    grads = torch.full((2 * N * (K + 1),), 7.0, device="cuda")
    c.layer(mrl).backward_gpu(ctx, None, grads, grad, x, c.params)
    ctx.synchronize()
    _, (want, off) = c.backward64()
    near(grads, want, off, "grads")
    del x, grad
    torch.cuda.empty_cache()
