"""A policy with a matrix memory as a user puts it together: a layer for all rows of the delta rule, the rule over a rollout with episode ends, a
gated feed-forward layer, a loss, the way back, clipping over all gradients, and an update by Muon and Adam."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


class Policy:
    """obs -> tanh layer -> [query | key | value | gate | rate] -> delta rule -> gated layer -> output layer, on device buffers."""

    def __init__(self, mrl, ctx, obs, hidden, heads, dk, dv, wide, out, steps, envs):
        self.mrl, self.ctx, self.steps, self.envs, rows = mrl, ctx, steps, envs, steps * envs
        self.rule, self.glu = mrl.GatedDeltaRule(heads, dk, dv), mrl.GatedLinear(heads * dv, wide, "silu")
        self.widths = [heads * dk, heads * dk, heads * dv, heads, heads]
        self.front = mrl.seq(mrl.LinearTanh(obs, hidden), mrl.Linear(hidden, sum(self.widths)))
        self.gates, self.back = mrl.Linear(heads * dv, 2 * wide), mrl.Linear(wide, out)
        opts = [mrl.Muon(self.front), mrl.Muon(self.gates, layers=[0]), mrl.Adam(lr=1e-3)]
        self.nets = [mrl.Network(ctx, m, o, mrl.Xavier(seed=k)) for k, (m, o) in enumerate(zip((self.front, self.gates, self.back), opts))]
        new = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        self.pre, self.h, self.f, self.out = new(rows, sum(self.widths)), new(rows, heads * dv), new(rows, wide), new(rows, out)
        self.caches = [new(rows * self.front.CACHE_SIZE), None, new(rows * self.back.CACHE_SIZE)]
        self.state, self.grad_state = new(envs, heads, dk, dv), new(envs, heads, dk, dv)
        self.grad_f, self.grad_h, self.grad_pre, self.grad_obs, self.norm = new(rows, wide), new(rows, heads * dv), new(rows, sum(self.widths)), new(rows, obs), new(1)

    def forward(self, obs, state, dones, prev, state_out=None):
        self.nets[0].forward_gpu(self.pre.view(-1), obs.view(-1), self.caches[0])
        self.rule.forward_gpu(self.ctx, self.h, *self.pre.split(self.widths, 1), self.steps, state_in=state, state_out=self.state if state_out is None else state_out, dones=dones, prev_dones=prev)
        self.glu.forward_gpu(self.ctx, self.f, self.h, self.nets[1].params)
        self.nets[2].forward_gpu(self.out.view(-1), self.f.view(-1), self.caches[2])

    def backward(self, grad_out, state, dones, prev, max_norm=None):
        self.nets[2].backward_gpu(self.grad_f.view(-1), grad_out.view(-1), self.caches[2])
        self.glu.backward_gpu(self.ctx, self.grad_h, self.nets[1].grads, self.grad_f, self.h, self.nets[1].params)
        self.rule.backward_gpu(self.ctx, *self.grad_pre.split(self.widths, 1), self.grad_h, *self.pre.split(self.widths, 1), self.steps, state_in=state, dones=dones,
                               prev_dones=prev, grad_state_in=self.grad_state)
        self.nets[0].backward_gpu(self.grad_obs.view(-1), self.grad_pre.view(-1), self.caches[0])
        if max_norm is not None:
            grads = [n.grads for n in self.nets]
            self.mrl.clip_grad_norm(self.ctx, grads, grads, max_norm, norm=self.norm)


def reference(policy, obs, state, cut, target):
    """The same in 64 bits with autograd: (outputs, parameter gradients, gradients of obs and state)."""
    front, gates, back = (n.params.cpu().double().requires_grad_() for n in policy.nets)
    obs, state = obs.cpu().double().requires_grad_(), state.cpu().double().requires_grad_()
    T, N, H = policy.steps, policy.envs, policy.rule.heads
    dk, dv = policy.rule.key_dim, policy.rule.value_dim

    def linear(x, params, a, b):
        return x @ params[:a * b].view(a, b) + params[a * b:a * b + b]
    (_, a, b), (_, c, d) = policy.front.layers
    x = torch.tanh(linear(obs, front[:a * b + b], a, b))
    pre = linear(x, front[a * b + b:], c, d)
    q, k, v, gate, rate = (t.reshape(T, N, H, -1) for t in pre.split(policy.widths, 1))
    q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    s, outs = state, []
    for t in range(T):
        s = torch.where(cut[t].view(N, 1, 1, 1), torch.zeros_like(s), s) * torch.sigmoid(gate[t]).unsqueeze(-1)
        u = torch.sigmoid(rate[t]).unsqueeze(-1) * (v[t].unsqueeze(2) - k[t].unsqueeze(2) @ s)
        s = s + k[t].unsqueeze(3) * u
        outs.append((q[t].unsqueeze(2) @ s).squeeze(2) / math.sqrt(dk))
    h = torch.stack(outs).reshape(T * N, H * dv)
    (_, e, f), = policy.gates.layers
    both = linear(h, gates, e, f)
    g, up = both[:, :f // 2], both[:, f // 2:]
    (_, i, j), = policy.back.layers
    out = linear(g * torch.sigmoid(g) * up, back, i, j)
    ((out - target.cpu().double()).square().sum() / 2).backward()
    return out.detach(), [front.grad, gates.grad, back.grad], obs.grad, state.grad


SHAPES = [(40, 6, 2, 16, 24, 48), (600, 2, 1, 64, 32, 100), (1, 64, 4, 24, 24, 32)]


def inputs(steps, envs, policy):
    gen = torch.Generator().manual_seed(steps)
    obs, target = torch.randn(steps * envs, 9, generator=gen).cuda(), torch.randn(steps * envs, 5, generator=gen).cuda()
    flags = (torch.rand(steps + 1, envs, generator=gen) < 0.05).float()
    state = torch.randn(policy.state.shape, generator=gen).cuda()
    return obs, target, state, flags[0].cuda(), flags[1:].contiguous().cuda(), flags[:-1] > 0.5


@pytest.mark.parametrize("steps,envs,heads,dk,dv,wide", SHAPES)
def test_training_step(mrl, ctx, steps, envs, heads, dk, dv, wide):
    policy = Policy(mrl, ctx, 9, 32, heads, dk, dv, wide, 5, steps, envs)
    obs, target, state, prev, dones, cut = inputs(steps, envs, policy)
    policy.forward(obs, state, dones, prev)
    grad_out = policy.out - target
    policy.backward(grad_out, state, dones, prev)
    ctx.synchronize()
    out, grads, grad_obs, grad_state = reference(policy, obs, state, cut, target)
    # fp32 products and sums of up to a few thousand terms in every layer: the 1e-4 that this suite allows the layers, in the 2-norm
    for got, want in ((policy.out, out), *zip([n.grads for n in policy.nets], grads), (policy.grad_obs, grad_obs), (policy.grad_state, grad_state)):
        got = got.cpu().double().reshape(want.shape)
        assert (got - want).norm() <= 1e-4 * want.norm() + 1e-9
    norm = torch.cat(grads).norm().item()
    policy.backward(grad_out, state, dones, prev, max_norm=norm / 3)
    ctx.synchronize()
    assert abs(policy.norm.item() - norm) <= 1e-4 * norm
    for net, want in zip(policy.nets, grads):
        assert (net.grads.cpu().double() * 3 - want).norm() <= 1e-4 * want.norm() + 1e-4 * want.norm()   # (the norm's share and its own)
    before = [n.params.clone() for n in policy.nets]
    for net in policy.nets:
        net.update_gpu()
    ctx.synchronize()
    for net, old in zip(policy.nets, before):
        step = (net.params - old).double()
        assert torch.isfinite(step).all() and (step * net.grads.double()).sum() < 0      # down the gradient


def test_collecting_step_by_step_is_the_rollout(mrl, ctx):
    """The states that single steps give while a rollout is collected are those of the training pass, across rollouts and episode ends."""
    steps, envs = 12, 33
    policy = Policy(mrl, ctx, 9, 16, 2, 20, 12, 40, 3, steps, envs)
    collect = Policy(mrl, ctx, 9, 16, 2, 20, 12, 40, 3, 1, envs)
    collect.nets = policy.nets
    state, prev = torch.zeros_like(policy.state), torch.zeros(envs, device="cuda")
    gen = torch.Generator().manual_seed(2)
    for rollout in range(3):
        first, first_prev = state.clone(), prev.clone()
        obs = torch.randn(steps * envs, 9, generator=gen).cuda()
        dones = (torch.rand(steps, envs, generator=gen) < 0.2).float().cuda()
        rows = []
        for t in range(steps):
            collect.forward(obs[t * envs:(t + 1) * envs].contiguous(), state, None, prev, state_out=state)
            rows.append(collect.out.clone())
            prev = dones[t]
        policy.forward(obs, first, dones, first_prev)
        ctx.synchronize()
        # outputs and states differ by what tiles of steps and another batch's layers may round differently
        assert (torch.cat(rows) - policy.out).abs().max() <= 1e-4 * policy.out.abs().max()
        assert (state - policy.state).abs().max() <= 1e-4 * policy.state.abs().max()


def test_the_whole_step_captured(mrl, ctx):
    """A training step in a graph, replayed on other observations with eager work between, gives what eager calls give."""
    side = torch.cuda.Stream()
    cctx = mrl.DeviceContext("cuda:0", stream=side)
    eager, captured = (Policy(mrl, c, 9, 32, 2, 24, 16, 48, 5, 50, 8) for c in (ctx, cctx))
    obs, target, state, prev, dones, _ = inputs(50, 8, eager)
    grad_out = torch.zeros_like(captured.out)
    captured.forward(obs, state, dones, prev)              # (the context makes room for the layers' sums at their first call, before a capture)
    captured.backward(grad_out, state, dones, prev, max_norm=0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured.forward(obs, state, dones, prev)
        torch.sub(captured.out, target, out=grad_out)
        captured.backward(grad_out, state, dones, prev, max_norm=0.5)
    for _ in range(4):
        obs.mul_(-0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.forward(obs, state, dones, prev)
        torch.cuda.synchronize()
        eager.backward(eager.out - target, state, dones, prev, max_norm=0.5)
        torch.cuda.synchronize()
        assert torch.equal(eager.out, captured.out) and torch.equal(eager.state, captured.state) and torch.equal(eager.norm, captured.norm)
        for a, b in zip(eager.nets, captured.nets):
            assert torch.equal(a.grads, b.grads)
        assert torch.equal(eager.grad_obs, captured.grad_obs) and torch.equal(eager.grad_state, captured.grad_state)
    del graph
    cctx.close()
