"""What GatedLinear refuses before anything reaches the library, on tensors of the host."""
import ctypes

import pytest
import torch


class HostContext:
    device, handle, stream = torch.device("cpu"), ctypes.c_void_p(), None


GOOD = dict(output=torch.zeros(6, 3), input=torch.zeros(6, 5), params=torch.zeros(36))


@pytest.mark.parametrize("bad,text", [
    (dict(input=torch.zeros(6, 4)), "input"), (dict(input=torch.zeros(30)), "input"), (dict(input=torch.zeros(6, 5, dtype=torch.float64)), "float32 or bfloat16"),
    (dict(output=torch.zeros(5, 3)), "output"), (dict(output=torch.zeros(6, 3, dtype=torch.bfloat16)), "output"), (dict(output=torch.zeros(3, 6).T), "next to each other"),
    (dict(params=torch.zeros(35)), "params"), (dict(params=torch.zeros(36, dtype=torch.bfloat16)), "params"), (dict(params=torch.zeros(72)[::2]), "params"),
    (dict(input=torch.zeros(5).expand(6, 5)), "overlap"), (dict(output=torch.zeros(6, 3).to("meta")), "output"),
])
def test_forward_refuses(mrl, bad, text):
    with pytest.raises(mrl.MrlError, match=text):
        mrl.GatedLinear(5, 3).forward_gpu(HostContext, **{**GOOD, **bad})


@pytest.mark.parametrize("bad,text", [(dict(grads=torch.zeros(36, dtype=torch.bfloat16)), "grads"), (dict(grads=torch.zeros(35)), "grads"), (dict(grad_input=torch.zeros(6, 4)), "grad_input"),
                                      (dict(grad_output=torch.zeros(6, 5)), "grad_output")])
def test_backward_refuses(mrl, bad, text):
    good = dict(grad_input=torch.zeros(6, 5), grads=torch.zeros(36), grad_output=torch.zeros(6, 3), input=torch.zeros(6, 5), params=torch.zeros(36))
    with pytest.raises(mrl.MrlError, match=text):
        mrl.GatedLinear(5, 3).backward_gpu(HostContext, **{**good, **bad})


def test_sizes_and_names(mrl):
    assert mrl.GatedLinear(5, 3).PARAM_SIZE == mrl.Linear(5, 6).PARAM_SIZE
    for args, text in (((0, 3), "dims"), ((5, 0), "dims"), ((5, 1 << 17), "dims"), ((5, 3, "relu6"), "activation")):
        with pytest.raises(mrl.MrlError, match=text):
            mrl.GatedLinear(*args)
    with pytest.raises(mrl.MrlError, match="2\\^26"):
        mrl.GatedLinear(5, 3).forward_gpu(HostContext, torch.empty(1 << 26, 3, device="meta"), torch.empty(1 << 26, 5, device="meta"), torch.zeros(36))
    for name, args in (("mrl_gated_linear_workspace", (None, 0, 1, 1, 1, 0, None)), ("mrl_gated_linear_forward", (None, 0, 0, 1, 1, 1, None, 1, None, None, 1, None, 0))):
        with pytest.raises(mrl.MrlError, match="ctx"):
            mrl._lib.call(name, *args)
