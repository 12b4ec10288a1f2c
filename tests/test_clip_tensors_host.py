"""What clip_grad_norm refuses before anything reaches the library, on tensors of the host."""
import ctypes

import pytest
import torch


class HostContext:
    device, handle, stream = torch.device("cpu"), ctypes.c_void_p(), None


@pytest.mark.parametrize("out,grads,max_norm,norm,text", [
    ([], [torch.zeros(3)], 1.0, None, "0 outputs for 1"), ([torch.zeros(4)], [torch.zeros(3)], 1.0, None, "does not fit"),
    ([torch.zeros(3, dtype=torch.bfloat16)], [torch.zeros(3)], 1.0, None, "does not fit"),
    ([torch.zeros(3, dtype=torch.float64)], [torch.zeros(3, dtype=torch.float64)], 1.0, None, "float32 or bfloat16"),
    ([torch.zeros(3, 2)], [torch.zeros(2, 3).T], 1.0, None, "grads\\[0\\] must be contiguous"), ([torch.zeros(2, 3).T], [torch.zeros(3, 2)], 1.0, None, "out\\[0\\] must be"),
    ([torch.zeros(3)], [torch.zeros(3)], -1.0, None, "max_norm"), ([torch.zeros(3)], [torch.zeros(3)], float("nan"), None, "max_norm"),
    ([torch.zeros(3)], [torch.zeros(3)], 1.0, torch.zeros(2), "norm"), ([torch.zeros(3)], [torch.zeros(3)], 1.0, torch.zeros(1, dtype=torch.float64), "norm"),
    ([torch.zeros(3, device="meta")], [torch.zeros(3)], 1.0, None, "out"), ([torch.zeros(3)], [torch.zeros(3)], 1.0, torch.zeros(1, device="meta"), "norm"),
])
def test_refuses(mrl, out, grads, max_norm, norm, text):
    with pytest.raises(mrl.MrlError, match=text):
        mrl.clip_grad_norm(HostContext, out, grads, max_norm, norm=norm)


def test_library_needs_a_context(mrl):
    with pytest.raises(mrl.MrlError, match="ctx"):
        mrl._lib.call("mrl_clip_tensors", None, 0, None, 1.0, None, None, 0)
