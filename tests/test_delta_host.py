"""What GatedDeltaRule refuses before anything reaches the library, on tensors of the host."""
import ctypes

import pytest
import torch


class HostContext:
    device, handle, stream = torch.device("cpu"), ctypes.c_void_p(), None


def layer(mrl):
    return mrl.GatedDeltaRule(4, 8, 6, key_heads=2)


def rows(**other):    # 3 steps of 2 environments
    z = torch.zeros
    return {**dict(query=z(6, 16), key=z(6, 16), value=z(6, 24), gate=z(6, 4), rate=z(6, 4), steps=3), **other}


BAD = [(dict(query=torch.zeros(6, 32)), "query"), (dict(key=torch.zeros(5, 16)), "key"), (dict(value=torch.zeros(6, 23)), "value"), (dict(value=torch.zeros(144)), "value"),
       (dict(value=torch.zeros(7, 24)), "value"), (dict(value=torch.zeros(6, 24, dtype=torch.float16)), "float32 or bfloat16"), (dict(gate=torch.zeros(6, 4, dtype=torch.bfloat16)), "gate"),
       (dict(rate=torch.zeros(6, 2)), "rate"), (dict(key=torch.zeros(16, 6).T), "next to each other"), (dict(query=torch.zeros(16).expand(6, 16)), "overlap"),
       (dict(steps=0), "steps"), (dict(steps=4), "steps"), (dict(dones=torch.zeros(5)), "dones"), (dict(prev_dones=torch.zeros(3)), "prev_dones"),
       (dict(state_in=torch.zeros(383)), "state_in"), (dict(state_in=torch.zeros(384, dtype=torch.bfloat16)), "state_in"), (dict(gate=torch.zeros(6, 4, device="meta")), "gate")]


@pytest.mark.parametrize("bad,text", BAD + [(dict(output=torch.zeros(6, 16)), "output"), (dict(output=torch.zeros(6, 24, dtype=torch.bfloat16)), "output"),
                                            (dict(state_out=torch.zeros(2, 4, 8, 5)), "state_out"), (dict(state_out=torch.zeros(768)[::2]), "state_out")])
def test_forward_refuses(mrl, bad, text):
    with pytest.raises(mrl.MrlError, match=text):
        layer(mrl).forward_gpu(HostContext, **{**rows(output=torch.zeros(6, 24)), **bad})


@pytest.mark.parametrize("bad,text", BAD + [(dict(grad_query=torch.zeros(6, 8)), "grad_query"), (dict(grad_key=torch.zeros(6, 16, dtype=torch.bfloat16)), "grad_key"),
                                            (dict(grad_value=torch.zeros(6, 16)), "grad_value"), (dict(grad_gate=torch.zeros(6, 2)), "grad_gate"),
                                            (dict(grad_rate=torch.zeros(4, 6).T), "next to each other"), (dict(grad_output=torch.zeros(6, 25)), "grad_output"),
                                            (dict(grad_state_out=torch.zeros(380)), "grad_state_out"), (dict(grad_state_in=torch.zeros(380)), "grad_state_in")])
def test_backward_refuses(mrl, bad, text):
    z = torch.zeros
    grads = dict(grad_query=z(6, 16), grad_key=z(6, 16), grad_value=z(6, 24), grad_gate=z(6, 4), grad_rate=z(6, 4), grad_output=z(6, 24))
    with pytest.raises(mrl.MrlError, match=text):
        layer(mrl).backward_gpu(HostContext, **{**rows(), **grads, **bad})


def test_sizes_and_null(mrl):
    made = layer(mrl)
    assert (made.key_width, made.value_width, made.state_size) == (16, 24, 192) and mrl.GatedDeltaRule(3, 5, 7).key_heads == 3
    for args, text in (((0, 8, 8), "heads"), ((4, 8, 8, 3), "heads"), ((4, 8, 8, 0), "heads"), ((4, 0, 8), "key_dim"), ((4, 129, 8), "key_dim"), ((4, 8, 0), "value_dim"),
                       ((4, 8, 129), "value_dim")):
        with pytest.raises(mrl.MrlError, match=text):
            mrl.GatedDeltaRule(*args)
    for name, args in (("mrl_delta_workspace", (None, None, 0, None)), ("mrl_delta_forward", (None, None, None, 0, None, None, 0)),
                       ("mrl_delta_backward", (None, None, None, 0, None, None, None, 0))):
        with pytest.raises(mrl.MrlError, match="NULL"):
            mrl._lib.call(name, *args)
