"""orthogonalize and Muon against the formulas in 64 bits."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


def polynomial(x, steps=5, eps=1e-7, gen=None):
    """In 64 bits; with `gen` every stored value off by what the kernels' arithmetic may cost it, at random: operands keep 22 bits (and
    2^-25 of a typical entry), a product's sum loses 2^-21 of the root of its terms' squares."""
    x = x.double()
    if x.shape[0] > x.shape[1]:
        return polynomial(x.T, steps, eps, gen).T

    def off(y, terms):
        typical = y.square().mean().sqrt()
        return y if gen is None else y + (2.0 ** -21 * terms + 2.0 ** -22 * y.abs() + 2.0 ** -25 * typical) * torch.randn(y.shape, generator=gen, dtype=torch.float64)

    def root(p, q):
        return ((p * p) @ (q * q)).sqrt() if gen is not None else None
    x = x / (x.norm() + eps)
    x = off(x, x.abs())
    for _ in range(steps):
        gram = off(x @ x.T, root(x, x.T))
        b = off(NS[1] * gram + NS[2] * (gram @ gram), 5 * gram.abs() + (2 * root(gram, gram) if gen is not None else 0))
        x = off(NS[0] * x + b @ x, 3.5 * x.abs() + (root(b, x) if gen is not None else 0))
    return x


def matrix(gen, rows, cols, rank=None):
    rank = rank or max(1, min(rows, cols) // 8)
    return torch.randn(rows, rank, generator=gen) @ torch.randn(rank, cols, generator=gen) / math.sqrt(rank) + 0.3 * torch.randn(rows, cols, generator=gen)


def near(got, x, half, what, steps=5, eps=1e-7):
    """Within eight times what the formula itself moves by when its intermediates are off as in polynomial(gen)."""
    want = polynomial(x, steps, eps)
    moved = (polynomial(x, steps, eps, torch.Generator().manual_seed(1)) - want).norm().item()
    off = (got.double().cpu() - want).norm().item()
    assert off <= 8 * moved + half * want.norm().item(), "%s: off by %g of %g, bound %g" % (what, off, want.norm(), 8 * moved + half * want.norm())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 50), (70, 1), (2, 2), (3, 4), (8, 256), (256, 4), (64, 64), (63, 65), (65, 63), (128, 128), (129, 127),
                                       (40, 600), (600, 40), (256, 256), (300, 777), (777, 333), (130, 1030), (513, 512), (1, 640), (33, 600), (96, 96), (97, 96), (64, 256), (257, 64)])
def test_orthogonalize(mrl, ctx, rows, cols, dtype):
    print("orthogonalize", rows, cols, dtype, flush=True)
    x = matrix(torch.Generator().manual_seed(rows * 1000 + cols), rows, cols).to(TYPES[dtype])
    out = torch.full((rows, cols), 9.0, dtype=TYPES[dtype], device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda())
    ctx.synchronize()
    near(out, x, HALF[dtype], "out")


@pytest.mark.parametrize("count,rows,cols,dtype", [(3, 30, 20, "f32"), (17, 9, 12, "bf16"), (40, 66, 70, "f32"), (2, 260, 100, "bf16"), (1, 5, 5, "f32")])
def test_many_matrices_in_place_at_odd_addresses(mrl, ctx, count, rows, cols, dtype):
    gen = torch.Generator().manual_seed(count)
    x = torch.stack([matrix(gen, rows, cols) * 10.0 ** (k % 5 - 2) for k in range(count)]).to(TYPES[dtype])
    flat = torch.full((x.numel() + 2,), -5.0, dtype=TYPES[dtype], device="cuda")
    inside = flat[1:-1].view(count, rows, cols)
    inside.copy_(x)
    mrl.orthogonalize(ctx, inside, inside)
    ctx.synchronize()
    assert flat[0] == -5 and flat[-1] == -5
    for k in range(count):
        near(inside[k], x[k], HALF[dtype], "matrix %d" % k)


# shapes whose products are worked out in larger tiles, alone and in batches, with rows and columns behind the last whole tile; batches
# in one launch, in one per product, and in more than one
@pytest.mark.parametrize("count,rows,cols,dtype", [(12, 519, 513, "f32"), (15, 449, 511, "bf16"), (8, 643, 701, "f32"), (60, 129, 191, "f32"), (6, 831, 385, "f32"),
                                                   (22, 193, 521, "bf16"), (1, 1411, 1500, "f32"), (5, 485, 2467, "f32"), (700, 20, 33, "f32"), (300, 65, 64, "bf16"), (650, 100, 130, "f32"), (14, 999, 1000, "bf16")])
def test_batches(mrl, ctx, count, rows, cols, dtype):
    print("batch", count, rows, cols, dtype, flush=True)
    gen = torch.Generator().manual_seed(count + rows)
    x = torch.randn(count, rows, cols, generator=gen)
    x[..., 0] += torch.arange(1.0, count + 1)[:, None] / count
    x = x.to(TYPES[dtype])
    out = torch.full((count, rows, cols), 9.0, dtype=TYPES[dtype], device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda())
    ctx.synchronize()
    for k in sorted({0, 1, 17, count // 2, 617, 618, count - 1}) if rows < 200 else {0, count - 1}:
        if k < count:
            near(out[k], x[k], HALF[dtype], "matrix %d" % k)
    norms = out.float().square().sum((1, 2)).cpu()
    # singular values of about [0.7, 1.2] have squares of 0.49 to 1.44; of random matrices' few start below the 1 / 485 that five steps lift
    assert (norms > 0.25 * min(rows, cols)).all() and (norms < 1.6 * min(rows, cols)).all()


@pytest.mark.parametrize("rows,cols", [(1, 500), (2, 300), (3, 50), (8, 64), (8, 721), (4, 1000), (14, 300), (16, 16), (2000, 12)])
def test_few_rows_as_close_as_fp32_products(mrl, ctx, rows, cols):
    """With few rows errors go one way in every entry: on average over matrices within twice what fp32 products are off (operands
    of 22 bits are rounded up to twice as far as those of 24)."""
    off, plain = 0.0, 0.0
    for seed in range(6):
        x = matrix(torch.Generator().manual_seed(100 + seed), rows, cols)
        out = torch.empty(rows, cols, device="cuda")
        mrl.orthogonalize(ctx, out, x.cuda())
        ctx.synchronize()
        want, y = polynomial(x), (x if rows <= cols else x.T) / (x.norm() + 1e-7)
        for _ in range(5):
            gram = y @ y.T
            y = NS[0] * y + (NS[1] * gram + NS[2] * gram @ gram) @ y
        off += ((out.cpu().double() - want).norm() / want.norm()).item()
        plain += (((y if rows <= cols else y.T).double() - want).norm() / want.norm()).item()
    print(rows, cols, off / 6, plain / 6, flush=True)
    assert off <= 2 * plain


@pytest.mark.parametrize("rows", [17, 20, 24, 33, 48, 64])
@pytest.mark.parametrize("cols", [64, 300, 1000])
def test_more_rows_as_close_as_fp32_products(mrl, ctx, rows, cols):
    """From 17 rows on products are taken on the fp16 cores: on average within twice what fp32 products are off, as those of fewer rows."""
    test_few_rows_as_close_as_fp32_products(mrl, ctx, rows, cols)


@pytest.mark.parametrize("steps,eps", [(1, 1e-7), (2, 1e-3), (3, 0.0), (8, 1e-7)])
def test_steps_and_eps(mrl, ctx, steps, eps):
    x = matrix(torch.Generator().manual_seed(steps), 48, 90) * 1e-3
    out = torch.empty(48, 90, device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda(), steps=steps, eps=eps)
    ctx.synchronize()
    near(out, x, HALF["f32"], "out", steps, eps)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 1e36])
def test_scales_near_the_ends_of_the_range(mrl, ctx, scale):
    """The norm is taken in 64 bits: neither its squares nor the quotient leave the range."""
    x = matrix(torch.Generator().manual_seed(3), 70, 50) * scale
    out = torch.empty(70, 50, device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda(), eps=0.0)
    ctx.synchronize()
    near(out, x, HALF["f32"], "out", eps=0.0)


def test_zeros_ones_and_what_is_not_finite(mrl, ctx):
    x = torch.zeros(4, 70, 90)
    x[1] = 1.0                      # one direction only
    x[2] = matrix(torch.Generator().manual_seed(1), 70, 90)
    x[2, 3, 4] = float("inf")
    x[3] = x[2]
    x[3, 3, 4] = float("nan")
    out = torch.empty_like(x, device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda())
    ctx.synchronize()
    assert not out[0].any() and torch.isnan(out[2]).all() and torch.isnan(out[3]).all()
    near(out[1], x[1], HALF["f32"], "ones")


@pytest.mark.parametrize("eps", [5e-324, 1e-310, 1e-300])
@pytest.mark.parametrize("rows,cols", [(4, 5), (130, 150)])
def test_zeros_with_the_least_eps(mrl, ctx, rows, cols, eps):
    """However small eps is above 0, zeros give zeros, and what is not zero is divided by its norm."""
    x = torch.zeros(2, rows, cols)
    x[1, 0, 0] = 2.0 ** -149
    out = torch.full_like(x, 9.0, device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda(), eps=eps)
    ctx.synchronize()
    assert not out[0].any()
    near(out[1], x[1], HALF["f32"], "the smallest", eps=eps)


def test_a_few_large_entries(mrl, ctx):
    """Entries at the top of the pieces' range, next to ones far below."""
    x = torch.randn(500, 700, generator=torch.Generator().manual_seed(2)) * 1e-4
    x[3, 5], x[100, 200] = 1.0, -0.7
    out = torch.empty(500, 700, device="cuda")
    mrl.orthogonalize(ctx, out, x.cuda())
    ctx.synchronize()
    near(out, x, HALF["f32"], "out")


def nets(mrl):
    return {
        "plain": mrl.seq(mrl.LinearReLU(8, 64), mrl.LinearReLU(64, 100), mrl.Linear(100, 4)),
        "gauss": mrl.seq(mrl.LinearTanh(17, 33), mrl.LinearTanh(33, 70), mrl.StochasticActor(70, 6)),
        "deep": mrl.seq(*[mrl.Linear(12, 12)] * 7, mrl.Linear(12, 300)),
        "one": mrl.Linear(5, 3),
    }


@pytest.mark.parametrize("net,layers,nesterov,decay", [("plain", None, True, 0.0), ("plain", (0, 1, 2), False, 0.1), ("plain", (), True, 0.0), ("plain", (1,), True, 0.5),
                                                       ("gauss", None, True, 0.01), ("gauss", (2,), True, 0.0), ("deep", None, False, 0.0),
                                                       ("deep", range(8), True, 0.0), ("one", None, True, 0.0), ("one", (0,), True, 0.0)])
def test_muon_steps(mrl, ctx, net, layers, nesterov, decay):
    print("muon", net, layers, nesterov, decay, flush=True)
    model = nets(mrl)[net]
    opt = mrl.Muon(model, lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=decay, layers=layers, adam_lr=1e-3, beta1=0.8, beta2=0.99, adam_eps=1e-6)
    n = model.PARAM_SIZE
    gen = torch.Generator().manual_seed(n)
    params, state = torch.randn(n, generator=gen), torch.zeros(2 * n)
    grads = [torch.randn(n, generator=gen) * 0.1 for _ in range(3)]
    p, s = params.cuda(), state.cuda()
    chosen = set(range(len(model.layers) - 1) if layers is None else layers)
    w, m2 = params.double(), state.double()
    loose = torch.zeros(n, dtype=torch.float64)       # what the products may move each parameter by
    for t, g in enumerate(grads, 1):
        opt.step_gpu(ctx, p, g.cuda(), s)
        g, at, adam = g.double(), 0, torch.ones(n, dtype=torch.bool)
        for k, (kind, rows, cols) in enumerate(model.layers):
            size = rows * cols
            if k in chosen:
                v = m2[2 * at:2 * at + size]
                v.mul_(0.9).add_(g[at:at + size])
                u = g[at:at + size] + 0.9 * v if nesterov else v
                o = polynomial(u.view(rows, cols))
                moved = (polynomial(u.view(rows, cols), gen=torch.Generator().manual_seed(t)) - o).norm().item()
                factor = 0.03 * max(1.0, cols / rows) ** 0.5
                w[at:at + size] = w[at:at + size] * (1 - 0.03 * decay) - factor * o.reshape(-1)
                loose[at:at + size] += factor * 8 * moved
                adam[at:at + size] = False
            at += size + (2 if kind == mrl.STOCHASTIC_ACTOR else 1) * cols
        assert at == n
        m, v = m2[0::2][adam], m2[1::2][adam]
        m, v = 0.8 * m + 0.2 * g[adam], 0.99 * v + 0.01 * g[adam] ** 2
        m2[0::2][adam], m2[1::2][adam] = m, v
        w[adam] -= 1e-3 * (m / (1 - 0.8 ** t)) / ((v / (1 - 0.99 ** t)).sqrt() + 1e-6)
    ctx.synchronize()
    assert opt.t == 3
    # a step rounds a parameter twice and its update (at most 0.003 by Adam, as many roundings as Adam has operations); the constants
    # 1 - beta, beta and the bias corrections are rounded to fp32
    bound = loose + 3 * (3 * 2.0 ** -24 * (w.abs() + 0.1) + 0.003 * 40 * 2.0 ** -24)
    assert ((p.cpu().double() - w).abs() <= bound).all()
    assert ((s.cpu().double() - m2).abs() <= 3 * 6 * 2.0 ** -24 * (m2.abs() + 0.5)).all()


# nets whose matrices take launches of their own for norms, products and update: tiles of 32 to 128, tall matrices, thin ones among
# large ones, unequal ones in one group
@pytest.mark.parametrize("widths,every,nesterov,decay", [((8, 256, 256, 4), False, True, 0.01), ((40, 700, 333, 900, 5), False, False, 0.1),
                                                         ((376, 1024, 1024, 1024, 17), True, True, 0.0), ((1500, 600, 11, 900), True, True, 0.05), ((2, 900, 900, 900), True, False, 0.3)])
def test_muon_steps_of_larger_nets(mrl, ctx, widths, every, nesterov, decay):
    print("muon", widths, every, nesterov, decay, flush=True)
    model = mrl.seq(*[mrl.LinearReLU(a, b) for a, b in zip(widths, widths[1:])])
    lr, mu, n, last = 0.03, 0.9, model.PARAM_SIZE, len(widths) - 2
    opt = mrl.Muon(model, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, layers=range(last + 1) if every else None, adam_lr=1e-3, beta1=0.8, beta2=0.99,
                   adam_eps=1e-6)
    gen = torch.Generator().manual_seed(sum(widths))
    params, state = 0.05 * torch.randn(n, generator=gen), torch.zeros(2 * n)
    shapes = list(zip(widths, widths[1:]))
    grads = [torch.cat([torch.cat((matrix(gen, a, b).reshape(-1), torch.randn(b, generator=gen))) for a, b in shapes]) for _ in range(2)]
    p, s = params.cuda(), state.cuda()
    w, m2 = params.double(), state.double()
    loose = [0.0] * len(shapes)       # what the products may move each matrix by, in the 2-norm
    for t, g in enumerate(grads, 1):
        opt.step_gpu(ctx, p, g.cuda(), s)
        g, at, adam = g.double(), 0, torch.ones(n, dtype=torch.bool)
        for k, (a, b) in enumerate(shapes):
            size = a * b
            if every or k < last:
                v = m2[2 * at:2 * at + size]
                v.mul_(mu).add_(g[at:at + size])
                u = (g[at:at + size] + mu * v if nesterov else v).view(a, b)
                o, factor = polynomial(u), lr * max(1.0, b / a) ** 0.5
                w[at:at + size] = w[at:at + size] * (1 - lr * decay) - factor * o.reshape(-1)
                loose[k] += factor * 8 * (polynomial(u, gen=torch.Generator().manual_seed(t)) - o).norm().item()
                adam[at:at + size] = False
            at += size + b
        m, v = m2[0::2][adam], m2[1::2][adam]
        m, v = 0.8 * m + 0.2 * g[adam], 0.99 * v + 0.01 * g[adam] ** 2
        m2[0::2][adam], m2[1::2][adam] = m, v
        w[adam] -= 1e-3 * (m / (1 - 0.8 ** t)) / ((v / (1 - 0.99 ** t)).sqrt() + 1e-6)
    ctx.synchronize()
    off, at = (p.cpu().double() - w), 0
    for k, (a, b) in enumerate(shapes):
        if every or k < last:
            # a step rounds a parameter at its product with the decay and at its update, and the constants 1 - lr decay and the factor
            here = slice(at, at + a * b)
            rounding = 2 * 2.0 ** -24 * (3 * w[here].norm().item() + 2 * lr * max(1.0, b / a) ** 0.5 * 1.3 * min(a, b) ** 0.5)
            assert off[here].norm().item() <= loose[k] + rounding, "matrix %d: %g, bound %g + %g" % (k, off[here].norm(), loose[k], rounding)
        at += a * b + b
    # Adam's share, element by element: an update of at most 0.003 of 40 roundings, a parameter rounded once, each of two steps
    assert (off[adam].abs() <= 2 * (2.0 ** -24 * (w[adam].abs() + 0.1) + 0.003 * 40 * 2.0 ** -24)).all()
    # gradients of up to 3 or so, a product and a sum rounded each step, constants rounded
    assert ((s.cpu().double() - m2).abs() <= 2 * 6 * 2.0 ** -24 * (m2.abs() + grads[0].abs().max() + 0.5)).all()


@pytest.mark.parametrize("large", [(), (3,), (30,)])
def test_more_matrices_than_a_launch_takes(mrl, ctx, large):
    """35 matrices with gaps between them in one call, against each in a call of its own."""
    lib, Matrix, gen = mrl._lib.lib(), mrl._lib.Matrix, torch.Generator().manual_seed(6)
    at, mats = 3, []
    for k in range(35):
        rows, cols = (150, 130) if k in large else (8 + k % 5, 12 - k % 3)
        mats.append(Matrix(at, rows, cols))
        at += rows * cols + k % 4
    n = at + 5
    p, g, s = torch.randn(n, generator=gen).cuda(), torch.randn(n, generator=gen).cuda(), torch.rand(2 * n, generator=gen).cuda()
    one = [p.clone(), g, s.clone()]
    ws = torch.empty(1 << 25, dtype=torch.uint8, device="cuda")

    def step(params, grads, state, matrices):
        array = (Matrix * max(1, len(matrices)))(*matrices)
        assert lib.mrl_muon_step(ctx.handle, *(ctypes.c_void_p(t.data_ptr()) for t in (params, grads, state)), params.numel(), len(matrices), array, 2, 0.1, 0.9, 1, 0.01, 5,
                                 1e-7, 1e-3, 0.9, 0.99, 1e-8, ctypes.c_void_p(ws.data_ptr()), ws.numel()) == 0, lib.mrl_last_error()
    step(p, g, s, mats)
    ctx.synchronize()
    start = 0
    for m in mats + [Matrix(n, 0, 0)]:
        end = m.offset + m.rows * m.cols
        step(one[0][start:end], g[start:end], one[2][2 * start:2 * end], [Matrix(m.offset - start, m.rows, m.cols)] if m.rows else [])
        ctx.synchronize()
        start = end
    assert torch.equal(s, one[2])
    # (a matrix in a launch of its own is worked out in other tiles: sums in another order, entries of at most 1.2 * 0.1 * sqrt(1.5))
    assert (p - one[0]).abs().max() <= 0.15 * 2.0 ** -14


def test_large_matrices_go_one_by_one(mrl, ctx):
    """Two matrices whose planes take more than a launch's share of a workspace: as each in a call of its own."""
    lib, Matrix, rows, cols = mrl._lib.lib(), mrl._lib.Matrix, 6000, 6100
    size, need = rows * cols, ctypes.c_uint64(0)
    mats = [Matrix(7, rows, cols), Matrix(size + 20, rows, cols)]
    assert lib.mrl_muon_workspace(2, (Matrix * 2)(*mats), ctypes.byref(need)) == 0
    n = 2 * size + 30
    torch.cuda.manual_seed(1)
    p, g, s = torch.randn(n, device="cuda"), torch.randn(n, device="cuda"), torch.zeros(2 * n, device="cuda")
    one, ws = [p.clone(), s.clone()], torch.empty(need.value, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def step(params, grads, state, matrices):
        array = (Matrix * len(matrices))(*matrices)
        assert lib.mrl_muon_step(ctx.handle, *(ctypes.c_void_p(t.data_ptr()) for t in (params, grads, state)), params.numel(), len(matrices), array, 1, 0.1, 0.9, 1, 0.0, 5,
                                 1e-7, 1e-3, 0.9, 0.99, 1e-8, ctypes.c_void_p(ws.data_ptr()), ws.numel()) == 0, lib.mrl_last_error()
    step(p, g, s, mats)
    step(one[0][:size + 20], g[:size + 20], one[1][:2 * size + 40], mats[:1])
    step(one[0][size + 20:], g[size + 20:], one[1][2 * size + 40:], [Matrix(0, rows, cols)])
    ctx.synchronize()
    assert torch.equal(p, one[0]) and torch.equal(s, one[1]) and p.isfinite().all()


@pytest.mark.parametrize("thin,others", [((9, 700), [(700, 700)] * 2), ((700, 9), [(700, 700)] * 2), ((8, 1024), [(1024, 1024)] * 2), ((16, 1000), [(1000, 1000)] * 3),
                                         ((1400, 16), [(900, 1400)]), ((5, 1500), [(1500, 1500)]), ((1, 900), [(600, 600)] * 6), ((2, 3000), [(2048, 2048)] * 2),
                                         ((4, 9000), [(2048, 2048)] * 2)])
def test_thin_matrix_does_not_go_by_its_neighbours(mrl, ctx, thin, others):
    """A matrix of up to 16 rows beside ones whose products are worked out in tiles of 64, 96 and 128: bit by bit what it is by itself, and as
    close to 64 bits as products in fp32."""
    print("thin", thin, others, flush=True)
    lib, Matrix, rows, cols = mrl._lib.lib(), mrl._lib.Matrix, *thin
    gen = torch.Generator().manual_seed(rows * cols)
    off = plain = 0.0
    large = torch.randn(sum(r * c for r, c in others), generator=gen).cuda()
    for seed in range(4):
        x = matrix(gen, rows, cols)
        grads = torch.cat((x.reshape(-1).cuda(), large))
        got = []
        for shapes in ([thin], [thin] + others):
            mats, at = [], 0
            for r, c in shapes:
                mats.append(Matrix(at, r, c))
                at += r * c
            array, need = (Matrix * len(mats))(*mats), ctypes.c_uint64(0)
            assert lib.mrl_muon_workspace(len(mats), array, ctypes.byref(need)) == 0
            ws, p, s = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda"), torch.zeros(at, device="cuda"), torch.zeros(2 * at, device="cuda")
            torch.cuda.synchronize()
            # momentum 0 and a rate of 1: the parameters become minus the polynomial, times the shape's factor
            assert lib.mrl_muon_step(ctx.handle, *(ctypes.c_void_p(t.data_ptr()) for t in (p, grads, s)), at, len(mats), array, 1, 1.0, 0.0, 0, 0.0, 5, 1e-7, 1e-3, 0.9, 0.99,
                                     1e-8, ctypes.c_void_p(ws.data_ptr()), ws.numel()) == 0, lib.mrl_last_error()
            ctx.synchronize()
            got.append(p[:rows * cols].cpu().view(rows, cols))
        assert torch.equal(*got)
        want, y = polynomial(x), (x if rows <= cols else x.T) / (x.norm() + 1e-7)
        for _ in range(5):
            gram = y @ y.T
            y = NS[0] * y + (NS[1] * gram + NS[2] * gram @ gram) @ y
        off += ((-got[1].double() / max(1.0, cols / rows) ** 0.5 - want).norm() / want.norm()).item()
        plain += (((y if rows <= cols else y.T).double() - want).norm() / want.norm()).item()
    # (operands of 22 bits are rounded up to twice as far as those of 24)
    assert off <= 2 * plain


@pytest.mark.parametrize("rows", [24, 64, 96])
def test_long_rows_cost_no_precision(mrl, ctx, rows):
    """The distance from 64 bits does not grow with the length of the rows: a sum is rounded in pieces of a fixed length, and joining eight
    of them adds about an eighth (in the root of the squares 1.06); the rest of the 1.5 is for the spread between matrices."""
    off = []
    for cols in (4096, 32768):
        total = 0.0
        for seed in range(6):
            gen = torch.Generator(device="cuda").manual_seed(300 + seed)
            rank = rows // 8
            x = torch.randn(rows, rank, device="cuda", generator=gen) @ torch.randn(rank, cols, device="cuda", generator=gen) / math.sqrt(rank)
            x += 0.5 * torch.randn(rows, cols, device="cuda", generator=gen)
            out = torch.empty_like(x)
            mrl.orthogonalize(ctx, out, x)
            want = polynomial(x)
            total += ((out.double() - want).norm() / want.norm()).item()
        off.append(total / 6)
    print(rows, off, flush=True)
    assert off[1] <= 1.5 * off[0]


def test_network_with_muon_trains_and_round_trips(mrl, ctx, tmp_path):
    """Behind Network as any optimiser: the parameters after update_gpu are those of the step on its own buffers, a checkpoint holds the momentum."""
    model = mrl.seq(mrl.LinearTanh(6, 48), mrl.LinearTanh(48, 48), mrl.Linear(48, 2))
    net = mrl.Network(ctx, model, mrl.Muon(model, lr=0.05), mrl.Xavier(seed=4))
    x, out, cache = torch.randn(32, 6, device="cuda"), torch.empty(64, device="cuda"), torch.empty(32 * model.CACHE_SIZE, device="cuda")
    net.forward_gpu(out, x.view(-1), cache)
    net.backward_gpu(torch.empty(192, device="cuda"), out.clone(), cache)
    params, state = net.params.clone(), net.optimizer_state.clone()
    other = mrl.Muon(model, lr=0.05)
    other.step_gpu(ctx, params, net.grads, state)
    net.update_gpu()
    ctx.synchronize()
    assert torch.equal(params, net.params) and torch.equal(state, net.optimizer_state) and state[:6 * 48].any()
    net.save_checkpoint(str(tmp_path / "net.txt"))
    again = mrl.Network(ctx, model, mrl.Muon(model), mrl.Xavier(seed=5))
    again.load_checkpoint(str(tmp_path / "net.txt"))
    assert torch.equal(again.params, net.params) and torch.equal(again.optimizer_state, net.optimizer_state)


def test_captured_graphs_keep_their_workspaces(mrl, ctx):
    gen = torch.Generator().manual_seed(8)
    xs = [matrix(gen, 200, 330).cuda(), matrix(gen, 330, 200).cuda()]
    wants = [torch.empty_like(x) for x in xs]
    for x, w in zip(xs, wants):
        mrl.orthogonalize(ctx, w, x)
    model = nets(mrl)["plain"]
    opt, n = mrl.Muon(model), model.PARAM_SIZE
    p0, g = torch.randn(n, generator=gen).cuda(), torch.randn(n, generator=gen).cuda()
    wp, ws = p0.clone(), torch.zeros(2 * n, device="cuda")
    mrl.Muon(model).step_gpu(ctx, wp, g, ws)
    ctx.synchronize()
    side = torch.cuda.Stream()
    cctx = mrl.DeviceContext("cuda:0", stream=side)
    graphs, outs = [], [torch.empty_like(x) for x in xs]
    p, s = p0.clone(), torch.zeros(2 * n, device="cuda")
    for x, o in zip(xs, outs):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            mrl.orthogonalize(cctx, o, x)
            if o is outs[0]:
                opt.step_gpu(cctx, p, g, s)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        p.copy_(p0)
        s.zero_()
        for o in outs:
            o.fill_(3)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        mrl.orthogonalize(ctx, torch.empty_like(xs[0]), xs[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants)) and torch.equal(p, wp) and torch.equal(s, ws)
    del graphs
    cctx.close()


def test_library_refusals(mrl, ctx):
    lib, size = mrl._lib.lib(), ctypes.c_uint64(0)
    assert lib.mrl_orthogonalize_workspace(1, 130, 8, ctypes.byref(size)) == 0 and size.value == 0
    x, y = torch.zeros(1 << 20, device="cuda"), torch.zeros(130 * 150, device="cuda")
    p, q = ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(y.data_ptr())
    assert lib.mrl_orthogonalize_workspace(1, 130, 150, ctypes.byref(size)) == 0 and 0 < size.value <= 1 << 22

    def orth(dtype=0, count=1, rows=130, cols=150, src=q, steps=5, eps=1e-7, ws=p, n=size.value):
        return lib.mrl_orthogonalize(ctx.handle, dtype, count, rows, cols, src, q, steps, eps, ws, n)
    for bad, text in ((dict(dtype=5), b"element type"), (dict(count=-1), b"count"), (dict(rows=0), b"sides"), (dict(cols=40000), b"sides"),
                      (dict(src=None), b"NULL"), (dict(steps=0), b"steps"), (dict(steps=65), b"steps"), (dict(eps=-1.0), b"eps"),
                      (dict(eps=float("nan")), b"eps"), (dict(n=size.value - 1), b"workspace holds"), (dict(ws=None), b"workspace holds"),
                      (dict(ws=ctypes.c_void_p(x.data_ptr() + 8)), b"aligned"), (dict(count=2), b"workspace holds")):
        assert orth(**bad) == -1 and text in lib.mrl_last_error(), bad
    Matrix = mrl._lib.Matrix

    def muon(mats=((0, 4, 4),), n=40000, t=1, steps=5, params=p, ws=p, size=1 << 18):
        array = (Matrix * max(1, len(mats)))(*[Matrix(*m) for m in mats])
        return lib.mrl_muon_step(ctx.handle, params, p, p, n, len(mats), array, t, 0.1, 0.9, 1, 0.0, steps, 1e-7, 1e-3, 0.9, 0.99, 1e-8, ws, size)
    for bad, text in ((dict(mats=((0, 4, 4), (15, 4, 4))), b"overlaps"), (dict(mats=((39990, 4, 4),)), b"overlaps"), (dict(mats=((-1, 4, 4),)), b"overlaps"),
                      (dict(mats=((0, 0, 4),)), b"sides"), (dict(n=-1), b"n <"), (dict(t=0), b"step count"), (dict(steps=0), b"steps"), (dict(params=None), b"NULL"),
                      (dict(mats=((0, 130, 150),), size=100), b"workspace holds")):
        assert muon(**bad) == -1 and text in lib.mrl_last_error(), bad
    ctx.synchronize()
    assert not x.any()


def test_buffers_that_overlap_are_refused(mrl, ctx):
    """Before anything is launched: they stay as they are."""
    x, model = torch.randn(8, 40, 30, device="cuda"), mrl.seq(mrl.Linear(6, 9), mrl.Linear(9, 3))
    n, before = model.PARAM_SIZE, x.clone()
    for out, src in ((x[1:], x[:-1]), (x[:-1], x[1:]), (x.view(-1)[1:2401].view(2, 40, 30), x[:2]), (x[3], x.view(-1)[3 * 1200 - 7:4 * 1200 - 7].view(40, 30))):
        with pytest.raises(mrl.MrlError, match="out and in overlap"):
            mrl.orthogonalize(ctx, out, src)
    flat, opt = x.view(-1), mrl.Muon(model)
    for p, g, s in ((flat[:n], flat[n - 1:2 * n - 1], flat[4000:4000 + 2 * n]), (flat[:n], flat[:n], flat[4000:4000 + 2 * n]), (flat[2 * n:3 * n], flat[4000:4000 + n], flat[n + 2 - n % 2:3 * n + 2 - n % 2]),
                    (flat[:n], flat[4000 + n:4000 + 2 * n], flat[4000:4000 + 2 * n])):
        with pytest.raises(mrl.MrlError, match="overlap"):
            opt.step_gpu(ctx, p, g, s)
    ctx.synchronize()
    assert opt.t == 0 and torch.equal(x, before)
    mrl.orthogonalize(ctx, x[1:], x[1:])         # in place, and next to each other
    mrl.orthogonalize(ctx, x[0], x[1])
    opt.step_gpu(ctx, flat[:n], flat[n:2 * n], flat[2 * n:4 * n])
    ctx.synchronize()
    # (the state was random numbers: below zero, its second moments have no square root)
    assert opt.t == 1 and flat[4 * n:].isfinite().all()
