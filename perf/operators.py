"""Timed cases of the operators of recurrent policies and of the matrix optimiser: the package's calls beside their plain forms.

  scan       GatedRecurrence.forward_gpu: a gated linear recurrence over a time-major rollout, cut where episodes end,
                 h[t] = a[t] * k[t] * h[t-1] + (1 - a[t]) * x[t],   a = sigmoid(gate),   k[t] = 0 where the step before ended an episode;
  scan_grad  GatedRecurrence.backward_gpu: the gradients of gate, value and first state from those of the outputs and the last state;
  step       GatedRecurrence.step_gpu: one step of every environment, the state updated in place;
  orth       orthogonalize: five Newton-Schulz steps X <- a X + (b A + c A A) X, A = X X^T, on matrices of Frobenius norm 1;
  muon       Muon.step_gpu: momentum, orthogonalisation and update of a network's hidden matrices, Adam for its other parameters.

Gates, values, outputs and matrices are float32 or bfloat16; states, momentum and parameters float32.  Everything is made from the
seed, on the device.  With `own` the package's kernels run, without it elementary torch operations in float32.
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
NS = (3.4445, -4.7750, 2.0315)      # the quintic's coefficients
MOST = 128 * 2048 * 256             # values of the largest rollout
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LR, MOMENTUM, DECAY, EPS = 0.02, 0.95, 0.01, 1e-7
ADAM_LR, BETA1, BETA2, ADAM_EPS = 3e-4, 0.9, 0.999, 1e-8


def listed():
    return [
        # a training pass over the rollout of many environments, gate and value the two halves of one layer's output rows
        dict(name="scan_rollout_2048", kind="scan", steps=128, envs=2048, width=256, dtype="f32", packed=True, dones=True),
        # a few long recorded sequences: little to do side by side, much along the time
        dict(name="scan_long_bf16", kind="scan", steps=16384, envs=2, width=512, dtype="bf16", packed=False, dones=True),
        # one odd-sized sequence of a small net
        dict(name="scan_odd_4097", kind="scan", steps=4097, envs=3, width=45, dtype="f32", packed=False, dones=False),
        # the same training pass backwards, half the environments
        dict(name="scan_grad_rollout_1024", kind="scan_grad", steps=128, envs=1024, width=256, dtype="f32", packed=True, dones=True),
        # a few long sequences backwards
        dict(name="scan_grad_long_bf16", kind="scan_grad", steps=8192, envs=4, width=320, dtype="bf16", packed=False, dones=True),
        # one step of the benchmark's 8192 environments while a rollout is collected
        dict(name="step_8192", kind="step", steps=1, envs=8192, width=256, dtype="f32", packed=True, dones=True),
        # one step of sixteen environments that live on the host: all latency
        dict(name="step_16_bf16", kind="step", steps=1, envs=16, width=64, dtype="bf16", packed=True, dones=True),
        # the hidden matrix of the benchmark's nets by itself
        dict(name="orth_256", kind="orth", count=1, rows=256, cols=256, dtype="f32"),
        # a wide net's hidden matrix
        dict(name="orth_2048", kind="orth", count=1, rows=2048, cols=2048, dtype="f32"),
        # several tall ragged matrices in bfloat16
        dict(name="orth_8x777x333_bf16", kind="orth", count=8, rows=777, cols=333, dtype="bf16"),
        # an update of the benchmark's actor: 8 inputs, two hidden layers of 256, 4 actions
        dict(name="muon_lunarlander", kind="muon", widths="8-256-256-4"),
        # a deep wide net: the hidden matrices are the work
        dict(name="muon_deep_1024", kind="muon", widths="376-1024-1024-1024-1024-17"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("scan", "scan", "scan_grad", "scan_grad", "step", "orth", "orth", "muon"))
    if kind == "orth":
        rows, cols, dtype = _log_int(rng, 4, 2048), _log_int(rng, 4, 2048), rng.choice(("f32", "bf16"))
        most = max(1, min(16, 2048 * 2048 // (rows * cols)))
        return dict(kind=kind, count=_log_int(rng, 1, most), rows=rows, cols=cols, dtype=dtype)
    if kind == "muon":
        hidden = [_log_int(rng, 16, 1024) for _ in range(rng.randint(2, 4))]
        widths = [_log_int(rng, 3, 400)] + hidden + [_log_int(rng, 1, 32)]
        return dict(kind=kind, widths="-".join(str(w) for w in widths))
    steps = 1 if kind == "step" else _log_int(rng, 1, 16384)
    width = _log_int(rng, 8, 1024)
    if rng.random() < 0.6:
        width = (width + 7) // 8 * 8    # most layers' widths are multiples of 8, some are odd
    room = min(MOST if kind == "scan" else MOST // 2, (8192 if kind == "step" else 1 << 17) * 256) // (steps * width)
    envs = _log_int(rng, 1, max(1, min(16384, room)))
    return dict(kind=kind, steps=steps, envs=envs, width=width, dtype=rng.choice(("f32", "bf16")), packed=rng.random() < 0.5,
                dones=rng.random() < 0.75)


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    s = dict(case)
    if case["kind"] == "orth":
        s["x"] = _gradients(randn, case["count"], case["rows"], case["cols"]).to(TYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["x"])
        return s
    if case["kind"] == "muon":
        widths = _widths(case)
        params, grads, state = [], [], []
        for i, (m, n) in enumerate(zip(widths, widths[1:])):
            params += [(randn(m * n + n) / math.sqrt(m))]
            grads += [_gradients(randn, 1, m, n).reshape(-1) * 1e-2, randn(n) * 1e-2]
            momentum = grads[-2] * 10 + randn(m * n) * 2e-2 if i < len(widths) - 2 else None
            first, second = randn(m * n + n) * 1e-2, randn(m * n + n).square() * 1e-4 + 1e-6
            moments = torch.stack((first, second), -1)
            if momentum is not None:        # a hidden matrix's share of the state starts with its momentum
                moments[:m * n] = torch.cat((momentum, torch.zeros_like(momentum))).view(m * n, 2)
            state += [moments.reshape(-1)]
        s.update(params=torch.cat(params), grads=torch.cat(grads), state=torch.cat(state), t=10)
        return s
    steps, envs, width, dtype = case["steps"], case["envs"], case["width"], TYPES[case["dtype"]]
    rows = steps * envs
    # gates with memories from a step to some hundreds of them, spread over the channels as trained ones are
    spread = torch.linspace(-1.0, 6.0, width, device=DEVICE)
    if case["packed"]:
        pre = torch.empty(rows, 2 * width, dtype=dtype, device=DEVICE)
        s["gate"], s["value"] = pre[:, :width], pre[:, width:]
    else:
        s["gate"], s["value"] = (torch.empty(rows, width, dtype=dtype, device=DEVICE) for _ in range(2))
    s["gate"].copy_(randn(rows, width) + spread)
    s["value"].copy_(randn(rows, width))
    s["hidden"] = randn(envs, width) * 0.5
    s["dones"] = s["prev_dones"] = None
    if case["dones"]:
        flags = (torch.rand(steps + 1, envs, device=DEVICE, generator=gen) < 0.01).float()
        s["prev_dones"], s["dones"] = flags[0].contiguous(), flags[1:].contiguous()
    s["out"] = torch.empty(rows, width, dtype=dtype, device=DEVICE)
    s["hidden_out"] = torch.empty(envs, width, device=DEVICE)
    if case["kind"] == "scan_grad":
        s["output"] = _scan(s)[0]
        s["grad_output"] = randn(rows, width).to(dtype)
        s["grad_hidden_out"] = randn(envs, width)
        s["grad_gate"], s["grad_value"] = torch.empty_like(s["out"]), torch.empty_like(s["out"])
        s["grad_hidden"] = torch.empty(envs, width, device=DEVICE)
    return s


def _gradients(randn, count, m, n):
    """Matrices as gradients are: a few strong directions over many weak ones."""
    rank = max(1, min(m, n) // 8)
    return 0.1 * (randn(count, m, rank) @ randn(count, rank, n) / math.sqrt(rank) + 0.5 * randn(count, m, n))


def _widths(case):
    return [int(w) for w in case["widths"].split("-")]


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
    if kind == "orth":
        mrl.orthogonalize(ctx, s["out"], s["x"], eps=EPS)
        return s["out"]
    if kind == "muon":
        if "optimizer" not in s:
            widths = _widths(s)
            hidden = [mrl.LinearReLU(m, n) for m, n in zip(widths[:-2], widths[1:-1])]
            s["optimizer"] = mrl.Muon(mrl.seq(*hidden, mrl.Linear(*widths[-2:])), lr=LR, momentum=MOMENTUM, weight_decay=DECAY, eps=EPS,
                                      adam_lr=ADAM_LR, beta1=BETA1, beta2=BETA2, adam_eps=ADAM_EPS)
            s["optimizer"].t = s["t"]
        s["optimizer"].step_gpu(ctx, s["params"], s["grads"], s["state"])
        return {"params": s["params"], "state": s["state"]}
    if "layer" not in s:
        s["layer"] = mrl.GatedRecurrence(s["width"])
    if kind == "step":
        s["layer"].step_gpu(ctx, s["out"], s["gate"], s["value"], s["hidden"], prev_dones=s["prev_dones"])
        return {"out": s["out"], "hidden": s["hidden"]}
    if kind == "scan":
        s["layer"].forward_gpu(ctx, s["out"], s["gate"], s["value"], s["steps"], state_in=s["hidden"], state_out=s["hidden_out"],
                               dones=s["dones"], prev_dones=s["prev_dones"])
        return {"out": s["out"], "hidden_out": s["hidden_out"]}
    s["layer"].backward_gpu(ctx, s["grad_gate"], s["grad_value"], s["grad_output"], s["gate"], s["value"], s["output"], s["steps"],
                            state_in=s["hidden"], dones=s["dones"], prev_dones=s["prev_dones"], grad_state_out=s["grad_hidden_out"],
                            grad_state_in=s["grad_hidden"])
    return {"gate": s["grad_gate"], "value": s["grad_value"], "hidden": s["grad_hidden"]}


# ---------------------------------------------------------------- plain forms


def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "orth":
        return _orthogonal(s["x"].float()).to(s["x"].dtype)
    if kind == "muon":
        return _muon(s)
    if kind == "step":
        a = torch.sigmoid(s["gate"].float())
        kept = s["hidden"] if s["prev_dones"] is None else torch.where(s["prev_dones"][:, None] > 0.5, 0.0, s["hidden"])
        s["hidden"].copy_(a * kept + torch.sigmoid(-s["gate"].float()) * s["value"].float())
        return {"out": s["hidden"].to(s["out"].dtype), "hidden": s["hidden"]}
    if kind == "scan":
        out, hidden = _scan(s)
        return {"out": out, "hidden_out": hidden}
    return _scan_grad(s)


def _by_step(s, x):
    return x.float().view(s["steps"], s["envs"], s["width"]) if x.is_contiguous() else x.float().reshape(s["steps"], s["envs"], s["width"])


def _keeps(s):
    """k[t] as [steps, envs, 1]: 0 where the step before ended an episode."""
    if s["dones"] is None:
        return torch.ones(s["steps"], s["envs"], 1, device=DEVICE)
    return (torch.cat((s["prev_dones"][None], s["dones"][:-1])) <= 0.5).float()[..., None]


def _linear_scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h = 0, by doubling: products and sums over 1, 2, 4, ... steps."""
    span = 1
    while span < len(a):
        b = torch.cat((b[:span], b[span:] + a[span:] * b[:-span]))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return b


def _scan(s):
    gate = _by_step(s, s["gate"])
    a = torch.sigmoid(gate) * _keeps(s)
    b = torch.sigmoid(-gate) * _by_step(s, s["value"])
    b[0] += a[0] * s["hidden"]
    h = _linear_scan(a, b)
    return h.view(s["steps"] * s["envs"], s["width"]).to(s["out"].dtype), h[-1].clone()


def _scan_grad(s):
    gate, keeps = _by_step(s, s["gate"]), _keeps(s)
    a = torch.sigmoid(gate)
    c = a * keeps
    grad = _by_step(s, s["grad_output"]).clone()
    grad[-1] += s["grad_hidden_out"]
    # grad[t] += c[t+1] * grad[t+1], from the last step to the first
    carried = torch.cat((c[1:], torch.zeros_like(c[:1])))
    grad = _linear_scan(carried.flip(0), grad.flip(0)).flip(0)
    before = torch.cat((s["hidden"][None], _by_step(s, s["output"])[:-1])) * keeps
    one_less = torch.sigmoid(-gate)
    flat = (s["steps"] * s["envs"], s["width"])
    grad_gate = a * one_less * (before - _by_step(s, s["value"])) * grad
    return {"gate": grad_gate.view(flat).to(s["out"].dtype), "value": (one_less * grad).view(flat).to(s["out"].dtype), "hidden": c[0] * grad[0]}


def _orthogonal(x):
    """[count, rows, cols] by five steps, on the side that has fewer rows."""
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = NS
    for _ in range(5):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _muon(s):
    widths = _widths(s)
    s["t"] += 1
    at = 0
    for i, (m, n) in enumerate(zip(widths, widths[1:])):
        size, hidden = m * n, i < len(widths) - 2
        if hidden:
            w, g, v = s["params"][at:at + size], s["grads"][at:at + size], s["state"][2 * at:2 * at + size]
            v.mul_(MOMENTUM).add_(g)
            o = _orthogonal((g + MOMENTUM * v).view(1, m, n)).view(-1)
            w.mul_(1 - LR * DECAY).sub_(LR * math.sqrt(max(1.0, n / m)) * o)
        rest = slice(at + size if hidden else at, at + size + n)
        w, g, mv = s["params"][rest], s["grads"][rest], s["state"][2 * rest.start:2 * rest.stop].view(-1, 2)
        mv[:, 0].mul_(BETA1).add_((1 - BETA1) * g)
        mv[:, 1].mul_(BETA2).add_((1 - BETA2) * g * g)
        w.sub_(ADAM_LR * (mv[:, 0] / (1 - BETA1 ** s["t"])) / ((mv[:, 1] / (1 - BETA2 ** s["t"])).sqrt() + ADAM_EPS))
        at += size + n
    return {"params": s["params"], "state": s["state"]}


# ---------------------------------------------------------------- the least work, and the definition in 64 bits


def work(case):
    if case["kind"] == "orth":
        one = _orthogonal_flops(case["rows"], case["cols"])
        values = case["count"] * case["rows"] * case["cols"]
        return {"bytes": 2 * values * (4 if case["dtype"] == "f32" else 2), "flops": case["count"] * one}
    if case["kind"] == "muon":
        widths = _widths(case)
        hidden = list(zip(widths[:-2], widths[1:-1]))
        matrices = sum(m * n for m, n in hidden)
        others = sum(hidden_n for _, hidden_n in hidden) + widths[-2] * widths[-1] + widths[-1]
        # parameters, momentum read and written, gradients read; for Adam both moments
        return {"bytes": 20 * matrices + 28 * others, "flops": sum(_orthogonal_flops(m, n) for m, n in hidden)}
    values, states = case["steps"] * case["envs"] * case["width"], case["envs"] * case["width"]
    size = 4 if case["dtype"] == "f32" else 2
    flags = 4 * case["steps"] * case["envs"] if case["dones"] else 0
    if case["kind"] == "scan_grad":
        return {"bytes": 6 * size * values + 12 * states + flags, "flops": 12 * values}
    return {"bytes": 3 * size * values + 8 * states + flags, "flops": 7 * values}


def _orthogonal_flops(rows, cols):
    """Five times a Gram matrix and a square, both symmetric, and the product with X."""
    m, n = min(rows, cols), max(rows, cols)
    return 5 * (m * m * n + m * m * m + 2 * m * m * n)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "orth":
        return torch.stack([_polynomial(m.double()) for m in s["x"]])
    if kind == "muon":
        params, state, t = s["params"].double(), s["state"].double(), s["t"] + 1
        grads, at = s["grads"].double(), 0
        widths = _widths(case)
        for layer in range(len(widths) - 1):
            m, n = widths[layer], widths[layer + 1]
            end = at + m * n
            if layer < len(widths) - 2:
                momentum = MOMENTUM * state[2 * at:2 * at + m * n] + grads[at:end]
                state[2 * at:2 * at + m * n] = momentum
                o = _polynomial((grads[at:end] + MOMENTUM * momentum).reshape(m, n)).reshape(-1)
                params[at:end] = params[at:end] * (1 - LR * DECAY) - LR * max(1.0, n / m) ** 0.5 * o
                at = end
            stop = end + n
            first = BETA1 * state[2 * at:2 * stop:2] + (1 - BETA1) * grads[at:stop]
            second = BETA2 * state[2 * at + 1:2 * stop:2] + (1 - BETA2) * grads[at:stop] ** 2
            state[2 * at:2 * stop:2], state[2 * at + 1:2 * stop:2] = first, second
            params[at:stop] -= ADAM_LR * (first / (1 - BETA1 ** t)) / ((second / (1 - BETA2 ** t)) ** 0.5 + ADAM_EPS)
            at = stop
        return {"params": params, "state": state}
    steps, envs, width = case["steps"], case["envs"], case["width"]
    shape = (steps, envs, width)
    gate, value = (s[k].double().reshape(shape) for k in ("gate", "value"))
    a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    cut = torch.zeros(steps, envs, 1, dtype=torch.bool, device=DEVICE)
    if s["prev_dones"] is not None:
        cut[0] = s["prev_dones"][:, None] > 0.5
        cut[1:] = s["dones"][:-1, :, None] > 0.5
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    if kind != "scan_grad":
        b, h, out = rest * value, s["hidden"].double(), torch.empty(shape, dtype=torch.float64, device=DEVICE)
        for t in range(steps):
            torch.addcmul(b[t], a[t], torch.where(cut[t], zero, h), out=out[t])
            h = out[t]
        return {"out": out.view(-1, width), "hidden" if kind == "step" else "hidden_out": h.clone()}
    c = torch.where(cut, zero, a)
    delta = s["grad_output"].double().reshape(shape).clone()
    delta[-1] += s["grad_hidden_out"].double()
    for t in range(steps - 2, -1, -1):
        delta[t].addcmul_(c[t + 1], delta[t + 1])
    before = torch.empty(shape, dtype=torch.float64, device=DEVICE)
    before[0], before[1:] = s["hidden"].double(), s["output"].double().reshape(shape)[:-1]
    before.masked_fill_(cut, 0.0)
    return {"gate": (delta * (before - value) * a * rest).view(-1, width), "value": (delta * rest).view(-1, width), "hidden": c[0] * delta[0]}


def _polynomial(x):
    """The same polynomial of the singular values from x's side with fewer rows, step by step in 64 bits."""
    if x.shape[0] > x.shape[1]:
        return _polynomial(x.T).T.contiguous()
    x = x / (torch.linalg.matrix_norm(x) + EPS)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(5):
        gram = x @ x.T
        x = (NS[0] * eye + gram @ (NS[1] * eye + NS[2] * gram)) @ x
    return x
