"""What GatedRecurrence refuses before anything reaches the library, on tensors of the host."""
import ctypes

import pytest
import torch


class HostContext:
    device, handle, stream = torch.device("cpu"), ctypes.c_void_p(), None


def rows(n=6, d=4, dtype=torch.float32):
    return torch.zeros(n, d, dtype=dtype)


GOOD = dict(output=rows(), gate=rows(), value=rows(), steps=3)


@pytest.mark.parametrize("bad,text", [
    (dict(steps=4), "steps"), (dict(steps=0), "steps"), (dict(gate=rows(6, 5)), "gate"), (dict(value=rows(5)), "value"),
    (dict(output=rows(dtype=torch.bfloat16)), "output"), (dict(gate=rows(dtype=torch.float64)), "float32 or bfloat16"),
    (dict(value=rows(4, 6).T), "next to each other"), (dict(output=torch.zeros(4).expand(6, 4)), "overlap"),
    (dict(state_in=torch.zeros(2, 5)), "state_in"), (dict(state_out=torch.zeros(2, 4, dtype=torch.bfloat16)), "state_out"),
    (dict(dones=torch.zeros(5)), "dones"), (dict(prev_dones=torch.zeros(3)), "prev_dones"), (dict(dones=torch.zeros(2, 3).T), "dones"),
    (dict(gate=torch.zeros(24)), "gate"), (dict(value=rows().to("meta")), "value"),
])
def test_forward_refuses(mrl, bad, text):
    with pytest.raises(mrl.MrlError, match=text):
        mrl.GatedRecurrence(4).forward_gpu(HostContext, **{**GOOD, **bad})


@pytest.mark.parametrize("name", ["grad_gate", "grad_value", "grad_output", "output"])
def test_backward_refuses(mrl, name):
    good = dict(grad_gate=rows(), grad_value=rows(), grad_output=rows(), gate=rows(), value=rows(), output=rows(), steps=2)
    with pytest.raises(mrl.MrlError, match=name):
        mrl.GatedRecurrence(4).backward_gpu(HostContext, **{**good, name: rows(6, 3)})
    for state in ("state_in", "grad_state_out", "grad_state_in"):
        with pytest.raises(mrl.MrlError, match=state):
            mrl.GatedRecurrence(4).backward_gpu(HostContext, **good, **{state: torch.zeros(4, 4)})


def test_width_and_context(mrl):
    with pytest.raises(mrl.MrlError, match="width"):
        mrl.GatedRecurrence(0)
    with pytest.raises(mrl.MrlError, match="ctx"):
        mrl.GatedRecurrence(4).forward_gpu(HostContext, **GOOD)
    for name, args in (("mrl_recurrence_workspace", (None, 1, 1, 1, None)),
                       ("mrl_recurrence_forward", (None, 0, 1, 1, 1, None, 1, None, 1, None, None, None, None, 1, None, None, 0))):
        with pytest.raises(mrl.MrlError, match="ctx"):
            mrl._lib.call(name, *args)


@pytest.mark.parametrize("rows,width,steps", [(1 << 32, 1, 1 << 32), (1 << 31, 1, 1), (1 << 20, 1 << 12, 1), (1 << 32, 2, 2)])
def test_more_than_the_library_counts(mrl, rows, width, steps):
    class Context:
        device, handle, stream = torch.device("meta"), ctypes.c_void_p(), None
    x = torch.empty(rows, width, device="meta")
    layer = mrl.GatedRecurrence(width)
    with pytest.raises(mrl.MrlError, match="2\\^31"):
        layer.forward_gpu(Context, x, x, x, steps)
    with pytest.raises(mrl.MrlError, match="2\\^31"):
        layer.backward_gpu(Context, x, x, x, x, x, x, steps)
