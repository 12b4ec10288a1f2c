"""A policy with memory as a user puts it together: layers, the recurrence over a rollout with episode ends, a loss, the way back, and
an update of its matrices by Muon."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(mrl):
    return mrl.DeviceContext("cuda:0")


class Policy:
    """obs -> tanh layer -> [gate | value] -> recurrence -> output layer, on device buffers."""

    def __init__(self, mrl, ctx, obs, hidden, width, out, steps, envs):
        self.ctx, self.width, self.steps, self.envs, rows = ctx, width, steps, envs, steps * envs
        self.front = mrl.seq(mrl.LinearTanh(obs, hidden), mrl.Linear(hidden, 2 * width))
        self.back = mrl.Linear(width, out)
        self.layer = mrl.GatedRecurrence(width)
        self.nets = [mrl.Network(ctx, m, mrl.Muon(m, lr=0.02, weight_decay=0.01, layers=range(len(m.layers))), mrl.Xavier(seed=k))
                     for k, m in enumerate((self.front, self.back))]
        new = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
        self.pre, self.h, self.out = new(rows, 2 * width), new(rows, width), new(rows, out)
        self.caches = [new(rows * m.CACHE_SIZE) for m in (self.front, self.back)]
        self.state, self.grad_state = new(envs, width), new(envs, width)
        self.grad_h, self.grad_pre, self.grad_obs = new(rows, width), new(rows, 2 * width), new(rows, obs)

    def forward(self, obs, state, dones, prev):
        w = self.width
        self.nets[0].forward_gpu(self.pre.view(-1), obs.view(-1), self.caches[0])
        self.layer.forward_gpu(self.ctx, self.h, self.pre[:, :w], self.pre[:, w:], self.steps, state_in=state, state_out=self.state, dones=dones,
                               prev_dones=prev)
        self.nets[1].forward_gpu(self.out.view(-1), self.h.view(-1), self.caches[1])

    def backward(self, grad_out, state, dones, prev):
        w = self.width
        self.nets[1].backward_gpu(self.grad_h.view(-1), grad_out.view(-1), self.caches[1])
        self.layer.backward_gpu(self.ctx, self.grad_pre[:, :w], self.grad_pre[:, w:], self.grad_h, self.pre[:, :w], self.pre[:, w:], self.h,
                                self.steps, state_in=state, dones=dones, prev_dones=prev, grad_state_in=self.grad_state)
        self.nets[0].backward_gpu(self.grad_obs.view(-1), self.grad_pre.view(-1), self.caches[0])


def reference(policy, obs, state, cut, target):
    """The same in 64 bits with autograd: (outputs, parameter gradients, gradients of obs and state)."""
    front, back = (n.params.cpu().double().requires_grad_() for n in policy.nets)
    obs, state = obs.cpu().double().requires_grad_(), state.cpu().double().requires_grad_()
    T, N, W = policy.steps, policy.envs, policy.width
    (_, a, b), (_, c, d) = policy.front.layers
    at = a * b
    x = torch.tanh(obs @ front[:at].view(a, b) + front[at:at + b])
    at += b
    pre = (x @ front[at:at + c * d].view(c, d) + front[at + c * d:]).view(T, N, 2 * W)
    gate, value = torch.sigmoid(pre[..., :W]), pre[..., W:]
    h, states = state, []
    for t in range(T):
        h = gate[t] * torch.where(cut[t][:, None], torch.zeros_like(h), h) + (1 - gate[t]) * value[t]
        states.append(h)
    (_, e, f), = policy.back.layers
    out = torch.cat(states) @ back[:e * f].view(e, f) + back[e * f:]
    ((out - target.cpu().double()).square().sum() / 2).backward()
    return out.detach(), (front.grad, back.grad), obs.grad, state.grad


@pytest.mark.parametrize("steps,envs,width", [(40, 6, 24), (600, 3, 40), (1, 64, 64)])
def test_training_step(mrl, ctx, steps, envs, width):
    torch.manual_seed(steps)
    policy = Policy(mrl, ctx, 9, 32, width, 5, steps, envs)
    obs, target, state = torch.randn(steps * envs, 9).cuda(), torch.randn(steps * envs, 5).cuda(), torch.randn(envs, width).cuda()
    flags = (torch.rand(steps + 1, envs) < 0.05).float()
    prev, dones = flags[0].cuda(), flags[1:].contiguous().cuda()
    policy.forward(obs, state, dones, prev)
    grad_out = policy.out - target
    policy.backward(grad_out, state, dones, prev)
    ctx.synchronize()
    out, grads, grad_obs, grad_state = reference(policy, obs, state, flags[:-1] > 0.5, target)
    # fp32 products and sums of up to a few thousand terms in every layer: the 1e-4 that this suite allows the layers, in the 2-norm
    for got, want in ((policy.out, out), (policy.nets[0].grads, grads[0]), (policy.nets[1].grads, grads[1]), (policy.grad_obs, grad_obs),
                      (policy.grad_state, grad_state)):
        got = got.cpu().double().reshape(want.shape)
        assert (got - want).norm() <= 1e-4 * want.norm() + 1e-9
    before = [n.params.clone() for n in policy.nets]
    for net in policy.nets:
        net.update_gpu()
    ctx.synchronize()
    for net, model, old in zip(policy.nets, (policy.front, policy.back), before):
        at = 0
        for _, rows, cols in model.layers:
            # an update's share of a matrix: singular values within [0.6, 1.3] of the step's length (five steps, from above 1e-2 of the
            # norm; smaller ones are still on their way up), so its 2-norm is at most 1.3 lr sqrt(max(1, cols / rows)) and not 0
            step = (net.params[at:at + rows * cols] - (1 - 0.02 * 0.01) * old[at:at + rows * cols]).view(rows, cols).double().cpu()
            top = torch.linalg.matrix_norm(step, 2).item() / (0.02 * max(1.0, cols / rows) ** 0.5)
            assert 0.6 <= top <= 1.3
            g = net.grads[at:at + rows * cols].view(rows, cols).double().cpu()
            assert (step * g).sum() < 0                 # down the gradient
            at += rows * cols + cols


def test_collecting_step_by_step_is_the_rollout(mrl, ctx):
    """The states that single steps give while a rollout is collected are those of the training pass, across rollouts and episode ends."""
    steps, envs, width = 12, 33, 20
    policy = Policy(mrl, ctx, 4, 16, width, 3, steps, envs)
    collect = Policy(mrl, ctx, 4, 16, width, 3, 1, envs)
    collect.nets = policy.nets
    state, prev = torch.zeros(envs, width, device="cuda"), torch.zeros(envs, device="cuda")
    gen = torch.Generator().manual_seed(2)
    for rollout in range(3):
        first, first_prev = state.clone(), prev.clone()
        obs = torch.randn(steps * envs, 4, generator=gen).cuda()
        dones = (torch.rand(steps, envs, generator=gen) < 0.2).float().cuda()
        rows = []
        for t in range(steps):
            collect.nets[0].forward_gpu(collect.pre.view(-1), obs[t * envs:(t + 1) * envs].reshape(-1))
            collect.layer.step_gpu(ctx, collect.h, collect.pre[:, :width], collect.pre[:, width:], state, prev_dones=prev)
            rows.append(collect.h.clone())
            prev = dones[t]
        policy.forward(obs, first, dones, first_prev)
        ctx.synchronize()
        # the states differ by what the scan's composed coefficients and another batch's layers may round differently
        scale = policy.h.abs().max().item()
        assert (torch.cat(rows) - policy.h).abs().max() <= 1e-4 * scale
        assert (state - policy.state).abs().max() <= 1e-4 * scale
