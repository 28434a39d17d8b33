"""Checks of forwards that wait for their backward (CSNet.set_train_checkpoints), shared by the emulator suite
(tests/test_waiting_emu.py) and the GPU suite (tests/test_gpu_waiting.py)."""
import pytest
import torch

import train_ops_cases as K
from oracle import inputs as I


def batch(seed, device, B=1, size=16):
    return torch.from_numpy(I.randn_batch(seed, B, size, size)).to(device)


def net(lib, device, manifest, act_dtype="fp32", fmt="int8", B=1):
    m = K._net(lib, device, manifest, act_dtype, B)
    m.set_train_checkpoints(fmt)
    return m


def grads(m):
    """All parameter gradients in one tensor; cleared on the way."""
    out = torch.cat([p.grad.reshape(-1) for p in m.parameters()]).clone()
    m.zero_grad(set_to_none=True)
    return out


def check_refilled_batch(lib, device, manifest, act_dtype):
    """One input buffer filled again for the next forward while the last one waits.  float32 steps read the batch again in their
    backward and refuse, the forward that is not waiting any more included; bfloat16 steps keep a copy and are right."""
    x = batch(31, device)
    m = net(lib, device, manifest, act_dtype)
    a, b = m(x), m(batch(32, device))
    dy = K.gradient(tuple(a.shape), torch.float32, 1, device)
    a.backward(dy)
    want = grads(m)
    m = net(lib, device, manifest, act_dtype)
    a = m(x)
    x.copy_(batch(32, device))
    b = m(x)
    if act_dtype == "bf16":
        a.backward(dy)
        assert torch.equal(grads(m), want)
    else:
        with pytest.raises(RuntimeError, match="image batch"):
            a.backward(dy)
        b.backward(dy)                       # (the newer forward has seen the buffer as it is)
        c = m(x)
        x.zero_()
        with pytest.raises(RuntimeError, match="image batch"):
            c.backward(dy)
