"""Timed cases of the operators of policies with a matrix memory: the package's calls beside their plain forms.

  delta       GatedDeltaRule.forward_gpu over a time-major rollout.  Per environment and head, with k = key / |key|,
              q = query / |query| / sqrt(key_dim), a = sigmoid(gate), b = sigmoid(rate),
                  S' = a[t] S[t-1] (0 where the step before ended an episode),  S[t] = S' + b[t] k[t] (v[t] - S'^T k[t])^T,  out[t] = S[t]^T q[t];
              |x| = sqrt(sum x^2 + 1e-6); groups of heads share a key head's query and key;
  delta_grad  GatedDeltaRule.backward_gpu: the gradients of query, key, value, gate, rate and first state;
  delta_step  GatedDeltaRule.step_gpu: one step of every environment, the state updated in place;
  glu         GatedLinear.forward_gpu: out = act(x Wg + bg) * (x Wu + bu), [Wg | Wu] the columns of one matrix;
  glu_grad    GatedLinear.backward_gpu: the gradients of x, the matrix and the biases;
  clip        clip_grad_norm over the gradients of several networks' parameter tensors: scaled so that the norm of all is at most max_norm.

Rows are float32 or bfloat16; states, the layers' parameter gradients and the norm are float32.  Everything is made from the seed, on the
device.  With `own` the package's kernels run, without it elementary torch operations in float32.
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
CHUNK = 64                          # steps that the plain form takes together, fewer where there are fewer
MOST = 128 * 1024 * 4 * 64 * 64     # multiply-adds of the largest rollout's state with one vector a step
GLU_MOST = 32768 * 512 * 2048
CLIP_MOST = 1 << 26


def listed():
    return [
        # a training pass over the rollout of many environments, everything in one layer's output rows
        dict(name="delta_rollout_1024", kind="delta", steps=128, envs=1024, heads=4, key_heads=4, key_dim=64, value_dim=64, dtype="f32", packed=True, dones=True),
        # two long recorded sequences with wide heads, two heads to a key head
        dict(name="delta_long_bf16", kind="delta", steps=8192, envs=2, heads=8, key_heads=4, key_dim=128, value_dim=128, dtype="bf16", packed=False, dones=True),
        # the training pass backwards, half the environments
        dict(name="delta_grad_rollout_512", kind="delta_grad", steps=128, envs=512, heads=4, key_heads=4, key_dim=64, value_dim=64, dtype="f32", packed=True, dones=True),
        # odd sizes backwards: a few sequences of a small net, three heads on one key head
        dict(name="delta_grad_odd_bf16", kind="delta_grad", steps=1001, envs=7, heads=3, key_heads=1, key_dim=40, value_dim=24, dtype="bf16", packed=False, dones=True),
        # one step of the benchmark's 8192 environments while a rollout is collected
        dict(name="delta_step_8192", kind="delta_step", steps=1, envs=8192, heads=4, key_heads=4, key_dim=64, value_dim=64, dtype="f32", packed=True, dones=True),
        # one step of sixteen environments that live on the host: all latency
        dict(name="delta_step_16_bf16", kind="delta_step", steps=1, envs=16, heads=2, key_heads=2, key_dim=32, value_dim=32, dtype="bf16", packed=True, dones=True),
        # sixteen rows through a wide layer: reading its matrix is the work
        dict(name="glu_16_rows", kind="glu", rows=16, in_dim=256, out_dim=1024, act="silu", dtype="f32"),
        # a large batch through a wide layer
        dict(name="glu_32768_bf16", kind="glu", rows=32768, in_dim=512, out_dim=2048, act="silu", dtype="bf16"),
        # the minibatch of an update of the benchmark's nets, an odd width
        dict(name="glu_grad_2048_f32", kind="glu_grad", rows=2048, in_dim=256, out_dim=683, act="gelu", dtype="f32"),
        # a large minibatch backwards
        dict(name="glu_grad_16384_bf16", kind="glu_grad", rows=16384, in_dim=512, out_dim=1024, act="silu", dtype="bf16"),
        # gradients of the benchmark's actor and critic: many small tensors
        dict(name="clip_lunarlander", kind="clip", nets="8-256-256-4,8-256-256-1", dtype="f32", max_norm=0.5),
        # two deep wide nets
        dict(name="clip_deep_2048", kind="clip", nets="376-2048-2048-2048-2048-17,376-2048-2048-2048-2048-1", dtype="f32", max_norm=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("delta", "delta", "delta_grad", "delta_grad", "delta_step", "glu", "glu", "glu_grad", "glu_grad", "clip"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "clip":
        nets, left = [], CLIP_MOST
        for _ in range(rng.randint(1, 4)):
            widths = [_log_int(rng, 3, 400)] + [_log_int(rng, 16, 4096) for _ in range(rng.randint(1, 5))] + [_log_int(rng, 1, 32)]
            left -= sum(m * n + n for m, n in zip(widths, widths[1:]))
            if left > 0:
                nets.append("-".join(str(w) for w in widths))
        nets = nets or ["%d-%d-%d" % (_log_int(rng, 3, 400), _log_int(rng, 16, 4096), _log_int(rng, 1, 32))]
        return dict(kind=kind, nets=",".join(nets), dtype=dtype, max_norm=rng.choice((0.5, 1.0, 1e6)))
    if kind in ("glu", "glu_grad"):
        in_dim, out_dim = _log_int(rng, 16, 2048), _log_int(rng, 16, 4096)
        if rng.random() < 0.6:
            in_dim, out_dim = (in_dim + 15) // 16 * 16, (out_dim + 15) // 16 * 16
        most = (GLU_MOST if kind == "glu" else GLU_MOST // 2) // (in_dim * out_dim) // (1 if dtype == "bf16" else 4)
        return dict(kind=kind, rows=_log_int(rng, 1, min(65536, max(1, most))), in_dim=in_dim, out_dim=out_dim,
                    act=rng.choice(("silu", "gelu", "sigmoid", "tanh")), dtype=dtype)
    key_heads, group = _log_int(rng, 1, 8), rng.choice((1, 1, 2, 3, 4))
    key_dim, value_dim = _log_int(rng, 8, 128), _log_int(rng, 8, 128)
    if rng.random() < 0.6:
        key_dim, value_dim = (key_dim + 15) // 16 * 16, (value_dim + 15) // 16 * 16
    heads = key_heads * group
    steps = 1 if kind == "delta_step" else _log_int(rng, 1, 8192)
    one = heads * max(key_dim, 16) * max(value_dim, 16)
    most = {"delta": MOST, "delta_grad": MOST // 2, "delta_step": 8192 * 4 * 64 * 64}[kind] // (steps * one)
    return dict(kind=kind, steps=steps, envs=_log_int(rng, 1, max(1, min(8192, most))), heads=heads, key_heads=key_heads, key_dim=key_dim,
                value_dim=value_dim, dtype=dtype, packed=rng.random() < 0.5, dones=rng.random() < 0.75)


# ---------------------------------------------------------------- inputs


def _tensors(case):
    """The shapes of the parameter tensors of the nets: a matrix and a bias for each layer."""
    shapes = []
    for net in case["nets"].split(","):
        widths = [int(w) for w in net.split("-")]
        for m, n in zip(widths, widths[1:]):
            shapes += [(m, n), (n,)]
    return shapes


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    s, dtype = dict(case), TYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "clip":
        s["grads"] = [(randn(*shape) * 1e-2).to(dtype) for shape in _tensors(case)]
        s["out"] = [torch.empty_like(g) for g in s["grads"]]
        s["norm"] = torch.empty(1, device=DEVICE)
        return s
    if kind in ("glu", "glu_grad"):
        rows, m, n = case["rows"], case["in_dim"], case["out_dim"]
        s["x"] = randn(rows, m).to(dtype)
        s["params"] = torch.cat((randn(m * 2 * n) / math.sqrt(m), randn(2 * n) * 0.1)).to(dtype)
        if kind == "glu":
            s["out"] = torch.empty(rows, n, dtype=dtype, device=DEVICE)
        else:
            s["grad_output"] = randn(rows, n).to(dtype)
            s["grad_x"] = torch.empty_like(s["x"])
            s["grads"] = torch.empty(m * 2 * n + 2 * n, device=DEVICE)
        return s
    steps, envs, heads, key_heads, dk, dv = (case[k] for k in ("steps", "envs", "heads", "key_heads", "key_dim", "value_dim"))
    rows = steps * envs
    widths = dict(query=key_heads * dk, key=key_heads * dk, value=heads * dv, gate=heads, rate=heads)
    if case["packed"]:
        parts = torch.empty(rows, sum(widths.values()), dtype=dtype, device=DEVICE).split(list(widths.values()), 1)
    else:
        parts = [torch.empty(rows, w, dtype=dtype, device=DEVICE) for w in widths.values()]
    # neighbouring keys are alike, as those of neighbouring observations are
    common = randn(envs, key_heads * dk).repeat(steps, 1)
    # memories from a step to some hundreds of them, spread over the heads as trained ones are
    spread = torch.linspace(0.0, 6.0, heads, device=DEVICE) if heads > 1 else 3.0
    for name, t in zip(widths, parts):
        x = randn(rows, t.shape[1])
        t.copy_(x + 0.7 * common if name == "key" else x + spread if name == "gate" else x)
        s[name] = t
    s["state"] = randn(envs, heads, dk, dv) * 0.3
    s["dones"] = s["prev_dones"] = None
    if case["dones"]:
        flags = (torch.rand(steps + 1, envs, device=DEVICE, generator=gen) < 0.01).float()
        s["prev_dones"], s["dones"] = flags[0].contiguous(), flags[1:].contiguous()
    if kind == "delta_grad":
        s["grad_output"] = randn(rows, heads * dv).to(dtype)
        s["grad_state_out"] = randn(envs, heads, dk, dv)
        s["grads"] = {name: torch.empty(rows, w, dtype=dtype, device=DEVICE) for name, w in widths.items()}
        s["grads"]["state"] = torch.empty_like(s["state"])
    else:
        s["out"] = torch.empty(rows, heads * dv, dtype=dtype, device=DEVICE)
        s["state_out"] = torch.empty_like(s["state"])
    return s


# ---------------------------------------------------------------- the package's calls

_made = {}


def _package():
    """The package and a context on the current stream, which a program makes once."""
    if not _made:
        import importlib
        _made["mrl"] = importlib.import_module("mojo-rl_amd")
        _made["ctx"] = _made["mrl"].DeviceContext("cuda:0")
    return _made["mrl"], _made["ctx"]


def _own(s):
    mrl, ctx = _package()
    kind = s["kind"]
    if kind == "clip":
        mrl.clip_grad_norm(ctx, s["out"], s["grads"], s["max_norm"], norm=s["norm"])
        return {"grads": s["out"], "norm": s["norm"]}
    if kind in ("glu", "glu_grad"):
        if "layer" not in s:
            s["layer"] = mrl.GatedLinear(s["in_dim"], s["out_dim"], s["act"])
        if kind == "glu":
            s["layer"].forward_gpu(ctx, s["out"], s["x"], s["params"])
            return s["out"]
        s["layer"].backward_gpu(ctx, s["grad_x"], s["grads"], s["grad_output"], s["x"], s["params"])
        return {"x": s["grad_x"], "params": s["grads"]}
    if "layer" not in s:
        s["layer"] = mrl.GatedDeltaRule(s["heads"], s["key_dim"], s["value_dim"], key_heads=s["key_heads"])
    rows = (s["query"], s["key"], s["value"], s["gate"], s["rate"])
    if kind == "delta_step":
        s["layer"].step_gpu(ctx, s["out"], *rows, s["state"], prev_dones=s["prev_dones"])
        return {"out": s["out"], "state": s["state"]}
    if kind == "delta":
        s["layer"].forward_gpu(ctx, s["out"], *rows, s["steps"], state_in=s["state"], state_out=s["state_out"], dones=s["dones"],
                               prev_dones=s["prev_dones"])
        return {"out": s["out"], "state": s["state_out"]}
    g = s["grads"]
    s["layer"].backward_gpu(ctx, g["query"], g["key"], g["value"], g["gate"], g["rate"], s["grad_output"], *rows, s["steps"],
                            state_in=s["state"], dones=s["dones"], prev_dones=s["prev_dones"], grad_state_out=s["grad_state_out"],
                            grad_state_in=g["state"])
    return g


# ---------------------------------------------------------------- plain forms


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "clip":
        norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / (norm + 1e-8), 1.0).float()
        return {"grads": [(g.float() * scale).to(g.dtype) for g in s["grads"]], "norm": norm.float().view(1)}
    if kind == "glu":
        gate, up = _pre(s)
        return (_act(s["act"], gate) * up).to(s["x"].dtype)
    if kind == "glu_grad":
        return _glu_grad(s)
    if kind == "delta_grad":
        return _delta_grad(s)
    rows = [s[name].float() for name in ("query", "key", "value", "gate", "rate")]
    out, state = _delta(s, rows, s["state"])
    if kind == "delta_step":
        s["state"].copy_(state)
        state = s["state"]
    return {"out": out.to(s["out"].dtype), "state": state}


def _weights(s):
    m, n = s["in_dim"], s["out_dim"]
    params = s["params"].float()
    return params[:m * 2 * n].view(m, 2 * n), params[m * 2 * n:]


def _pre(s):
    w, b = _weights(s)
    return (s["x"].float() @ w + b).split(s["out_dim"], 1)


def _act(act, g):
    if act == "tanh":
        return torch.tanh(g)
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return torch.sigmoid(g) * (g if act == "silu" else 1)


def _act_grad(act, g):
    if act == "tanh":
        return 1 - torch.tanh(g).square()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    a, rest = torch.sigmoid(g), torch.sigmoid(-g)
    return a * (1 + g * rest) if act == "silu" else a * rest


def _glu_grad(s):
    gate, up = _pre(s)
    x, w, grad = s["x"].float(), _weights(s)[0], s["grad_output"].float()
    pre = torch.cat((grad * up * _act_grad(s["act"], gate), grad * _act(s["act"], gate)), 1)
    return {"x": (pre @ w.t()).to(s["x"].dtype), "params": torch.cat(((x.t() @ pre).view(-1), pre.sum(0)))}


def _unit_lower_inverse(m):
    """The inverse of unit lower triangular matrices, their sides a power of two, from blocks of one row to blocks of all."""
    side = m.shape[-1]
    out = torch.eye(side, device=m.device).expand(m.shape)
    block = torch.arange(side, device=m.device)
    size = 1
    while size < side:
        # the inverse of [[P, 0], [R, Q]] is [[P', 0], [-Q' R P', Q']]
        of, pair = block // size, block // (2 * size)
        below = ((of[:, None] > of[None]) & (pair[:, None] == pair[None])).float()
        out = out - out @ (m * below) @ out
        size *= 2
    return out


def _delta(s, rows, state):
    """Outputs and last states of all steps, up to CHUNK of them at a time: within a chunk S[t] is the state ahead of it and a sum over the
    chunk's steps, each with u = b (v - S'^T k), and the u solve a unit lower triangular system."""
    steps, envs, heads, dk, dv = s["steps"], s["envs"], s["heads"], s["key_dim"], s["value_dim"]
    chunk = min(CHUNK, 1 << (steps - 1).bit_length())
    chunks = (steps + chunk - 1) // chunk
    more = chunks * chunk - steps

    def by_chunk(x, share):
        """[rows, parts * width] as [envs * heads, chunks, chunk, width]; steps behind the last one are zeros"""
        x = x.reshape(steps, envs, share, -1).permute(1, 2, 0, 3).repeat_interleave(heads // share, 1)
        return torch.cat((x, x.new_zeros(envs, heads, more, x.shape[3])), 2).reshape(envs * heads, chunks, chunk, -1)

    def unit(x):
        return x / (x.square().sum(-1, keepdim=True) + EPS).sqrt()

    q = by_chunk(rows[0], s["key_heads"])
    q, k, v = unit(q) / math.sqrt(dk), unit(by_chunk(rows[1], s["key_heads"])), by_chunk(rows[2], heads)
    there = by_chunk(torch.ones(steps * envs, heads, device=DEVICE), heads)
    b = by_chunk(torch.sigmoid(rows[4]), heads) * there
    # sums of logarithms in 64 bits: differences of long ones are wanted
    log_a = by_chunk(-torch.logaddexp(-rows[3].double(), rows[3].double().new_zeros(())), heads)
    cut = torch.zeros_like(log_a)
    if s["dones"] is not None:
        cut = by_chunk(torch.cat((s["prev_dones"][None], s["dones"][:-1])).view(-1, 1).expand(-1, heads).double().gt(0.5).double(), heads)
    since = (log_a * (1 - cut)).cumsum(2)
    episode = cut.cumsum(2)
    same = (episode == episode.transpose(2, 3)).float()
    lower = torch.ones(chunk, chunk, device=DEVICE).tril()
    decay = torch.exp((since - since.transpose(2, 3)) * lower).float() * lower * same
    first = torch.exp(since).float() * (episode == 0)
    last = torch.exp(since[:, :, -1:] - since).float() * (episode == episode[:, :, -1:])
    keys = k @ k.transpose(2, 3)
    solve = _unit_lower_inverse(torch.eye(chunk, device=DEVICE) + b * keys * decay * lower.tril(-1))
    u0, w = solve @ (b * v), solve @ (b * first * k)
    inside, outside = (q @ k.transpose(2, 3)) * decay, q * first
    onto, kept = (k * last).transpose(2, 3), first[:, :, -1:]
    state, outs = state.reshape(envs * heads, dk, dv), []
    for c in range(chunks):
        u = u0[:, c] - w[:, c] @ state
        outs.append(outside[:, c] @ state + inside[:, c] @ u)
        state = kept[:, c] * state + onto[:, c] @ u
    out = torch.cat(outs, 1)[:, :steps].reshape(envs, heads, steps, dv).permute(2, 0, 1, 3).reshape(steps * envs, heads * dv)
    return out, state.view(envs, heads, dk, dv)


def _delta_grad(s):
    names = ("query", "key", "value", "gate", "rate")
    with torch.enable_grad():
        rows = [s[name].float().requires_grad_() for name in names]
        state = s["state"].clone().requires_grad_()
        found = torch.autograd.grad(_delta(s, rows, state), [*rows, state], [s["grad_output"].float(), s["grad_state_out"]])
    return {**{name: g.to(s[name].dtype) for name, g in zip(names, found)}, "state": found[5]}


# ---------------------------------------------------------------- the least work, and the definition in 64 bits


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind == "clip":
        values = sum(math.prod(shape) for shape in _tensors(case))
        return {"bytes": 2 * size * values, "flops": 3 * values}
    if kind in ("glu", "glu_grad"):
        rows, m, n = case["rows"], case["in_dim"], case["out_dim"]
        params = 2 * n * (m + 1)
        if kind == "glu":
            return {"bytes": size * (rows * (m + n) + params), "flops": 4 * rows * m * n}
        return {"bytes": size * (rows * (2 * m + n) + params) + 4 * params, "flops": 12 * rows * m * n}
    steps, envs, heads, key_heads, dk, dv = (case[k] for k in ("steps", "envs", "heads", "key_heads", "key_dim", "value_dim"))
    rows, states = steps * envs, envs * heads * dk * dv
    read = 2 * key_heads * dk + heads * dv + 2 * heads
    flags = 4 * rows if case["dones"] else 0
    if kind == "delta_grad":
        return {"bytes": size * rows * (2 * read + heads * dv) + 12 * states + flags, "flops": 20 * rows * heads * dk * dv}
    return {"bytes": size * rows * (read + heads * dv) + 8 * states + flags, "flops": 7 * rows * heads * dk * dv}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        total = sum(float((g.double() ** 2).sum()) for g in s["grads"])
        norm = total ** 0.5
        scale = case["max_norm"] / (norm + 1e-8) if norm > case["max_norm"] else 1.0
        return {"grads": [g.double() * scale for g in s["grads"]], "norm": torch.tensor([norm], dtype=torch.float64, device=DEVICE)}
    if kind in ("glu", "glu_grad"):
        return _exact_glu(s)
    return _exact_delta(s)


def _exact_glu(s):
    m, n = s["in_dim"], s["out_dim"]
    p, x = s["params"].double(), s["x"].double()
    columns = p[:m * 2 * n].view(m, 2, n)
    gate, up = (x @ columns[:, i].contiguous() + p[m * 2 * n + i * n:m * 2 * n + (i + 1) * n] for i in (0, 1))
    sig = 1 / (1 + torch.exp(-gate))
    bell, phi = torch.exp(-gate ** 2 / 2) / (2 * math.pi) ** 0.5, torch.special.ndtr(gate)
    value, slope = {"sigmoid": (sig, sig * (1 - sig)), "silu": (gate * sig, sig + gate * sig * (1 - sig)), "gelu": (gate * phi, phi + gate * bell),
                    "tanh": (2 / (1 + torch.exp(-2 * gate)) - 1, 4 * torch.exp(-2 * gate) / (1 + torch.exp(-2 * gate)) ** 2)}[s["act"]]
    if s["kind"] == "glu":
        return value * up
    grad = s["grad_output"].double()
    parts = grad * up * slope, grad * value
    grads = torch.stack([x.t() @ part for part in parts], 1)
    return {"x": sum(part @ columns[:, i].t() for i, part in enumerate(parts)), "params": torch.cat([grads.reshape(-1)] + [part.sum(0) for part in parts])}


def _exact_delta(s):
    steps, envs, heads, key_heads, dk, dv = (s[k] for k in ("steps", "envs", "heads", "key_heads", "key_dim", "value_dim"))
    group = heads // key_heads
    q, k = (s[name].double().reshape(steps, envs, key_heads, 1, dk).expand(-1, -1, -1, group, -1).reshape(steps, envs, heads, dk) for name in ("query", "key"))
    v = s["value"].double().reshape(steps, envs, heads, dv)
    a, b = (1 / (1 + torch.exp(-s[name].double())).reshape(steps, envs, heads, 1, 1) for name in ("gate", "rate"))
    q_len, k_len = ((x.square().sum(-1, keepdim=True) + EPS).sqrt() for x in (q, k))
    q, k = q / q_len, k / k_len
    if s["dones"] is not None:
        cut = torch.cat((s["prev_dones"][None], s["dones"][:-1])) > 0.5
        a = torch.where(cut.view(steps, envs, 1, 1, 1), 0.0, a)
    grad = s["kind"] == "delta_grad"
    state = s["state"].double().reshape(envs, heads, dk, dv)
    before = torch.empty(steps, *state.shape, dtype=torch.float64, device=DEVICE) if grad else None
    out = torch.empty(steps, envs, heads, dv, dtype=torch.float64, device=DEVICE)
    for t in range(steps):
        if grad:
            before[t] = state
        state = a[t] * state
        u = b[t] * (v[t].unsqueeze(2) - k[t].unsqueeze(2) @ state)
        state = state + k[t].unsqueeze(3) * u
        out[t] = (q[t].unsqueeze(2) @ state).squeeze(2) / dk ** 0.5
    if not grad:
        return {"out": out.view(steps * envs, -1), "state": state}
    d_out = s["grad_output"].double().reshape(steps, envs, heads, dv) / dk ** 0.5
    d_state = s["grad_state_out"].double()
    found = {name: torch.empty_like(x) for name, x in (("query", q), ("key", k), ("value", v), ("gate", a), ("rate", b))}
    for t in range(steps - 1, -1, -1):
        kept = a[t] * before[t]
        kt, go = k[t].unsqueeze(3), d_out[t].unsqueeze(2)
        miss = v[t].unsqueeze(2) - k[t].unsqueeze(2) @ kept
        found["query"][t] = ((kept + kt * (b[t] * miss)) @ go.transpose(2, 3)).squeeze(3)
        d_state = d_state + q[t].unsqueeze(3) * go
        pulled = kt.transpose(2, 3) @ d_state
        found["value"][t] = (b[t] * pulled).squeeze(2)
        found["rate"][t] = (pulled * miss).sum((2, 3), keepdim=True) * b[t] * (1 - b[t])
        found["key"][t] = (b[t] * (d_state @ miss.transpose(2, 3) - kept @ pulled.transpose(2, 3))).squeeze(3)
        d_state = d_state - kt * (b[t] * pulled)
        found["gate"][t] = (d_state * kept).sum((2, 3), keepdim=True) * (1 - a[t])
        d_state = a[t] * d_state
    for name, x, length in (("query", q, q_len), ("key", k, k_len)):
        g = found[name]
        g = (g - x * (x * g).sum(-1, keepdim=True)) / length
        found[name] = g.view(steps, envs, key_heads, group, dk).sum(3)
    return {**{name: g.reshape(steps * envs, -1) for name, g in found.items()}, "state": d_state}
