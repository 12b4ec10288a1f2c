"""What orthogonalize and Muon refuse before anything reaches the device, and the shares of the flat parameters that Muon takes."""
import ctypes

import pytest
import torch


class HostContext:
    device, handle, stream = torch.device("cpu"), ctypes.c_void_p(), None


@pytest.mark.parametrize("x,out,text", [
    (torch.zeros(4), torch.zeros(4), "rows, cols"), (torch.zeros(2, 2, 2, 2), torch.zeros(2, 2, 2, 2), "rows, cols"),
    (torch.zeros(3, 4, dtype=torch.float64), torch.zeros(3, 4, dtype=torch.float64), "float32 or bfloat16"),
    (torch.zeros(3, 4), torch.zeros(4, 3), "does not fit"), (torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.bfloat16), "does not fit"),
    (torch.zeros(4, 3).T, torch.zeros(3, 4), "contiguous"), (torch.zeros(3, 4), torch.zeros(4, 3).T, "contiguous"),
    (torch.zeros(3, 4, device="meta"), torch.zeros(3, 4), "on cpu expected"),
])
def test_orthogonalize_refuses(mrl, x, out, text):
    with pytest.raises(mrl.MrlError, match=text):
        mrl.orthogonalize(HostContext, out, x)


@pytest.mark.parametrize("shape", [(1 << 31, 1, 1), (2, (1 << 32) + 5), (1, (1 << 32) + 5, 2)])
def test_more_than_the_library_counts(mrl, shape):
    class Context:
        device, handle, stream = torch.device("meta"), ctypes.c_void_p(), None
    with pytest.raises(mrl.MrlError, match="counts"):
        mrl.orthogonalize(Context, torch.empty(shape, device="meta"), torch.empty(shape, device="meta"))


def test_nothing_to_do_needs_no_device(mrl):
    for shape in ((0, 4), (4, 0), (0, 3, 4)):
        mrl.orthogonalize(HostContext, torch.zeros(shape), torch.zeros(shape))


def test_muon_shares(mrl):
    model = mrl.seq(mrl.LinearReLU(8, 256), mrl.LinearTanh(256, 64), mrl.StochasticActor(64, 4))

    def shares(**kw):
        opt = mrl.Muon(model, **kw)
        return [(m.offset, m.rows, m.cols) for m in opt._matrices[:opt._count]]
    second = 8 * 256 + 256
    third = second + 256 * 64 + 64
    assert shares() == [(0, 8, 256), (second, 256, 64)]
    assert shares(layers=(2, 0)) == [(0, 8, 256), (third, 64, 4)] and shares(layers=()) == []
    assert mrl.Muon(model).STATE_PER_PARAM == 2 and mrl.Muon(model).t == 0
    for bad in ((3,), (-1,)):
        with pytest.raises(mrl.MrlError, match="layers"):
            mrl.Muon(model, layers=bad)


def test_muon_step_refuses(mrl):
    model = mrl.seq(mrl.Linear(4, 6), mrl.Linear(6, 2))
    n, opt = model.PARAM_SIZE, mrl.Muon(model)
    for p, g, s, text in ((n - 1, n, 2 * n, "params"), (n, n + 1, 2 * n, "grads"), (n, n, n, "state")):
        with pytest.raises(mrl.MrlError, match=text):
            opt.step_gpu(HostContext, torch.zeros(p), torch.zeros(g), torch.zeros(s))
    with pytest.raises(mrl.MrlError, match="params"):
        opt.step_gpu(HostContext, torch.zeros(n, dtype=torch.bfloat16), torch.zeros(n), torch.zeros(2 * n))
    assert opt.t == 0


def test_null_contexts_and_workspace_queries(mrl):
    size = ctypes.c_uint64(0)
    mrl._lib.call("mrl_orthogonalize_workspace", 3, 400, 340, ctypes.byref(size))
    assert size.value >= 3 * (6 * 2 * 340 * 400 + 4 * 2 * 340 * 340)
    mrl._lib.call("mrl_orthogonalize_workspace", 3, 40, 30, ctypes.byref(size))
    assert size.value == 0   # (held in LDS)
    mrl._lib.call("mrl_orthogonalize_workspace", 1, 1 << 15, 1 << 15, ctypes.byref(size))
    one = size.value
    mrl._lib.call("mrl_orthogonalize_workspace", 1000, 1 << 15, 1 << 15, ctypes.byref(size))
    assert size.value == one   # (a large matrix fills the device by itself)
    Matrix = mrl._lib.Matrix
    large = (Matrix * 20)(*[Matrix(k << 30, 1 << 15, 1 << 15) for k in range(20)])
    mrl._lib.call("mrl_muon_workspace", 20, large, ctypes.byref(size))
    assert size.value == one
    mrl._lib.call("mrl_muon_workspace", 0, None, ctypes.byref(size))
    assert size.value == 0
    for name, args in (("mrl_orthogonalize", (None, 0, 1, 4, 4, None, None, 5, 1e-7, None, 0)),
                       ("mrl_muon_step", (None, None, None, None, 4, 0, None, 1, 0.1, 0.9, 1, 0.0, 5, 1e-7, 1e-3, 0.9, 0.99, 1e-8, None, 0))):
        with pytest.raises(mrl.MrlError, match="ctx"):
            mrl._lib.call(name, *args)
    for args in ((1, 0, 4), (-1, 4, 4), (1, 4, 1 << 16)):
        with pytest.raises(mrl.MrlError):
            mrl._lib.call("mrl_orthogonalize_workspace", *args, ctypes.byref(size))


def test_ppo_update_refuses_what_is_not_adam(mrl):
    """The update's kernels apply Adam with the optimiser's lr, beta1, beta2 and eps, which mean something else in Muon."""
    actor = mrl.seq(mrl.LinearReLU(4, 64), mrl.LinearReLU(64, 64), mrl.Linear(64, 2))
    critic = mrl.seq(mrl.LinearReLU(4, 64), mrl.LinearReLU(64, 64), mrl.Linear(64, 1))
    rb = mrl.ppo.RolloutBuffers(HostContext, mrl.CartPoleEnv, actor, critic, 5, 3)
    for cls in (mrl.ppo.PPOUpdate, mrl.ppo.DiscreteUpdate, mrl.ppo.ContinuousUpdate):
        for opts in ((mrl.Muon(actor), mrl.Muon(critic)), (mrl.Muon(actor), mrl.Adam()), (mrl.Adam(), mrl.Muon(critic))):
            with pytest.raises(mrl.MrlError, match="cannot run Muon"):
                cls(HostContext, rb, 4, *opts)

    class Mine(mrl.Adam):
        pass
    upd = mrl.ppo.PPOUpdate(HostContext, rb, 4, Mine(lr=0.1), mrl.Adam(lr=0.2))
    upd.actor_opt = mrl.Muon(actor)          # (put in place of the first one later)
    with pytest.raises(mrl.MrlError, match="cannot run Muon"):
        upd.minibatch_step(torch.zeros(4, dtype=torch.int32))
    assert upd.actor_opt.t == 0 and upd.critic_opt.t == 0


def test_agent_with_muon_networks_refuses_to_train(mrl):
    agent = mrl.DeepPPOAgent(obs_dim=4, num_actions=2, hidden_dim=64, n_envs=4, rollout_len=8, gpu_minibatch_size=16)
    am, cm = agent._nets()
    net = lambda model: type("Net", (), dict(model=model, params=torch.zeros(model.PARAM_SIZE), optimizer=mrl.Muon(model)))  # noqa: E731
    agent.actor, agent.critic = net(am), net(cm)
    with pytest.raises(mrl.MrlError, match="cannot run Muon"):
        agent._build(HostContext, mrl.CartPoleEnv)
