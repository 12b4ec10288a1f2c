"""clip_grad_norm over many tensors against 64 bits."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# The sum of squares is exact to far below a unit of fp32; the factor is rounded once and the product once: 2 units.  bf16 is rounded once
# more, by up to 2^-8.
OFF = {torch.float32: 2.5 * UNIT, torch.bfloat16: 2.0 ** -8 + 3 * UNIT}


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


def tensors(sizes, dtypes, scale=1e-2, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(TYPES[dtypes[i % len(dtypes)]]).cuda() for i, n in enumerate(sizes)]


def check(mrl, ctx, grads, max_norm, out):
    host = [g.cpu().double() for g in grads]
    want_norm = sum(float((g ** 2).sum()) for g in host) ** 0.5
    scale = max_norm / (want_norm + 1e-8) if want_norm > max_norm else 1.0
    norm = torch.full((1,), 7.0, device="cuda")
    mrl.clip_grad_norm(ctx, out, grads, max_norm, norm=norm)
    ctx.synchronize()
    if want_norm < 3.4e38:
        assert abs(norm.item() - want_norm) <= 1.5 * UNIT * want_norm
    else:
        assert norm.item() == float("inf")   # what fp32 rounds it to; the factor is taken from the Float64 norm
    for o, g in zip(out, host):
        got = o.cpu().double()
        if scale == 1.0:
            assert torch.equal(got, g)
        else:
            # (below 2^-126 fp32 goes in steps of 2^-149)
            assert ((got - g * scale).abs() <= OFF[o.dtype] * (g * scale).abs() + 2.0 ** -149).all()


@pytest.mark.parametrize("place", ["in", "out"])
@pytest.mark.parametrize("max_norm", [0.01, 0.5, 1e6])
@pytest.mark.parametrize("sizes,dtypes", [((1,), ("f32",)), ((7, 1, 0, 9), ("f32", "bf16")), ((2047, 2048, 2049, 8, 3), ("bf16",)), ((100000, 33, 70000), ("f32",)),
                                          (tuple(range(1, 250)), ("f32", "bf16")), ((5000001, 17), ("f32",)), ((3,) * 96, ("f32",)), ((3,) * 97, ("bf16",))])
def test_against_64_bits(mrl, ctx, sizes, dtypes, max_norm, place):
    print("clip", len(sizes), max(sizes), dtypes, max_norm, place, flush=True)
    grads = tensors(sizes, dtypes)
    check(mrl, ctx, grads, max_norm, grads if place == "in" else [torch.full_like(g, 7.0) for g in grads])


def test_at_any_alignment(mrl, ctx):
    flat = tensors([100000], ["f32"])[0]
    half = flat.to(torch.bfloat16)
    grads = [flat[1:30002], half[1:40004], half[50001:50002], flat[30003:99999]]
    check(mrl, ctx, grads, 0.3, [torch.empty_like(g) for g in grads])
    before = flat.clone()
    mrl.clip_grad_norm(ctx, grads, grads, 0.3)
    ctx.synchronize()
    assert flat[0] == before[0] and flat[30002] == before[30002] and flat[99999] == before[99999]   # neighbours stay as they were


def test_the_ends_of_the_range(mrl, ctx):
    big = torch.full((1000,), 3e38, device="cuda")
    small = torch.full((1000,), 1e-30, device="cuda")
    check(mrl, ctx, [big, small], 2.0, [torch.empty_like(big), torch.empty_like(small)])
    check(mrl, ctx, [small], 1e-40, [torch.empty_like(small)])     # squares that fp32 does not hold
    norm, out = torch.empty(1, device="cuda"), torch.empty(2, device="cuda")
    mrl.clip_grad_norm(ctx, [out], [torch.tensor([float("inf"), 1.0], device="cuda")], 1.0, norm=norm)
    ctx.synchronize()
    assert norm.item() == float("inf") and torch.isnan(out[0]) and out[1] == 0
    mrl.clip_grad_norm(ctx, [out], [torch.tensor([float("nan"), 1.0], device="cuda")], 0.1, norm=norm)
    ctx.synchronize()
    assert torch.isnan(norm).all() and torch.isnan(out[0]) and out[1] == 1
    norm.fill_(7.0)
    mrl.clip_grad_norm(ctx, [], [], 1.0, norm=norm)
    ctx.synchronize()
    assert norm.item() == 0.0


def test_same_as_the_flat_call(mrl, ctx):
    """the parts of one vector, clipped together, against ppo.clip_grad_norm of the vector: sums in another order and precision"""
    flat = tensors([70000], ["f32"])[0]
    parts = [p.clone() for p in flat.split([30000, 1, 39999])]
    mrl.clip_grad_norm(ctx, parts, parts, 0.5)
    mrl.ppo.clip_grad_norm(ctx, flat, 0.5)
    ctx.synchronize()
    # (the flat call sums 70000 squares in fp32, at most 300 of them one behind the other in a partial sum)
    assert ((torch.cat(parts) - flat).abs() <= 300 * UNIT * flat.abs()).all()


def test_captured_and_replayed(mrl, ctx):
    stream = torch.cuda.Stream()
    side = mrl.DeviceContext("cuda:0", stream=stream)
    grads = tensors((5000, 3, 40000), ("f32",))
    out, norm = [torch.empty_like(g) for g in grads], torch.empty(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        mrl.clip_grad_norm(side, out, grads, 0.5, norm=norm)
    for i in range(3):
        for g in grads:
            g.mul_(1.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager, eager_norm = [torch.empty_like(g) for g in grads], torch.empty(1, device="cuda")
        mrl.clip_grad_norm(ctx, eager, grads, 0.5, norm=eager_norm)
        torch.cuda.synchronize()
        assert torch.equal(norm, eager_norm) and all(torch.equal(a, b) for a, b in zip(out, eager))
    side.close()


def test_library_refuses(mrl, ctx):
    x = torch.zeros(64, device="cuda")
    ws = torch.empty(mrl._lib.CLIP_TENSORS_WORKSPACE, dtype=torch.uint8, device="cuda")

    def call(entries, workspace=ws.data_ptr(), size=mrl._lib.CLIP_TENSORS_WORKSPACE, norm=None):
        mrl._lib.call("mrl_clip_tensors", ctx.handle, len(entries), (mrl._lib.Tensor * len(entries))(*entries), 1.0, norm, workspace, size)
    at = x.data_ptr()
    for entries, text in (([(at, at + 4, 8, 0)], "overlap"), ([(at, at, 8, 0), (at, at, 8, 0)], "overlap"), ([(at, at, 8, 0), (at + 64, at + 16, 8, 0)], "overlap"),
                          ([(at, at + 128, 8, 0), (at + 132, at + 64, 4, 0)], "overlap"), ([(at, at, -1, 0)], "values"), ([(at, at, 8, 5)], "type"),
                          ([(None, at, 8, 0)], "NULL")):
        with pytest.raises(mrl.MrlError, match=text):
            call(entries)
    good = [(at, at, 8, 0)]
    for kwargs, text in ((dict(size=100), "workspace"), (dict(workspace=None), "workspace"), (dict(workspace=ws.data_ptr() + 4), "aligned"), (dict(norm=at), "norm"),
                         (dict(norm=ws.data_ptr()), "overlap")):
        with pytest.raises(mrl.MrlError, match=text):
            call(good, **kwargs)
    call([(at, at + 64, 8, 0), (at, at + 128, 8, 0)])   # the same input twice is fine
    ctx.synchronize()


def test_a_tensor_past_2_to_the_31(mrl, ctx):
    n = (1 << 31) + 4099
    big, small = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.full((3,), 2.0, device="cuda")
    big[-1], big[1 << 31], big[5] = 8.0, 4.0, 2.0
    norm = torch.empty(1, device="cuda")
    mrl.clip_grad_norm(ctx, [big, small], [big, small], 2.0, norm=norm)
    ctx.synchronize()
    length = (64.0 + 16 + 4 + 12) ** 0.5
    assert abs(norm.item() - length) <= 1.5 * UNIT * length
    got = torch.stack([big[-1], big[1 << 31], big[5], *small]).double().cpu()
    want = torch.tensor([8.0, 4.0, 2.0, 2.0, 2.0, 2.0], dtype=torch.float64) * 2 / length
    assert ((got - want).abs() <= OFF[torch.bfloat16] * want).all() and torch.count_nonzero(big).item() == 3


@pytest.mark.parametrize("max_norm", [-1.0, float("nan")])
def test_library_refuses_a_norm_below_0(mrl, ctx, max_norm):
    x, ws = torch.ones(8, device="cuda"), torch.empty(mrl._lib.CLIP_TENSORS_WORKSPACE, dtype=torch.uint8, device="cuda")
    entries = (mrl._lib.Tensor * 1)((x.data_ptr(), x.data_ptr(), 8, 0))
    with pytest.raises(mrl.MrlError, match="max_norm"):
        mrl._lib.call("mrl_clip_tensors", ctx.handle, 1, entries, max_norm, None, ws.data_ptr(), mrl._lib.CLIP_TENSORS_WORKSPACE)
    ctx.synchronize()
    assert (x == 1).all()
