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


def check_two_streams(lib, device, manifest, act_dtype, B, size, rounds):
    """Forward a on one stream, forward b on another that waits for it, one backward over both: autograd runs b's node on b's stream and
    a's on a's, with no wait between them.  The gradients are those of one stream."""
    xs = [batch(s, device, B, size) for s in (31, 32)]
    dy = K.gradient((B, 1, size, size), torch.float32, 1, device)
    m = net(lib, device, manifest, act_dtype, B=B)
    a, b = (m(x) for x in xs)
    torch.autograd.backward([a, b], [dy, dy])
    want = grads(m)
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    for _ in range(rounds):
        m = net(lib, device, manifest, act_dtype, B=B)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            a = m(xs[0])
        streams[1].wait_stream(streams[0])
        with torch.cuda.stream(streams[1]):
            b = m(xs[1])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.autograd.backward([a, b], [dy, dy])
        torch.cuda.synchronize()
        assert torch.equal(grads(m), want)


def check_changed_parameters(lib, device, manifest):
    """Parameters that something other than a torch operation on them changes while a forward waits: the fused optimizer's step and a
    model that was moved are refused, before and after the forward was displaced; a write through ``.data``, which leaves no trace,
    changes nothing: the gradients are those of the forward's parameters."""
    from sod100k_amd.tools.train import FusedTrainer
    x, other = batch(31, device), batch(32, device)
    dy = K.gradient((1, 1, 16, 16), torch.float32, 1, device)
    m = net(lib, device, manifest)
    m(x).backward(dy)
    exact = grads(m)
    a, b = m(x), m(other)
    a.backward(dy)
    kept = grads(m)
    del b

    m = net(lib, device, manifest)
    tr = FusedTrainer(m, lr=1e-2, lib=lib)
    a = m(x)
    tr.step(other, torch.zeros(1, 1, 16, 16, device=device))
    with pytest.raises(RuntimeError, match="in-place change"):
        a.backward(dy)
    m = net(lib, device, manifest)
    a = m(x)
    m._apply(lambda t: t)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="in-place change"):
            a.backward(dy)
        m.eval()(x)                          # (there is an arena again, another one)
        m.train()
    for displaced, want in ((False, exact), (True, kept)):
        m = net(lib, device, manifest)
        a = m(x)
        for p in m.parameters():
            p.data.mul_(1.5)
        if displaced:
            b = m(other)
        a.backward(dy)
        assert torch.equal(grads(m), want)


def check_failed_save(lib, device, manifest):
    """The checkpoint that would make room for the next forward cannot be had (out of memory): that forward raises and the one that
    waits keeps its place, exact gradients included; so it does where an older forward's backward wanted the room."""
    xs = [batch(s, device) for s in (31, 32)]
    dy = K.gradient((1, 1, 16, 16), torch.float32, 1, device)
    m = net(lib, device, manifest)
    m(xs[1]).backward(dy)
    exact = grads(m)
    eng = m.engine_for(xs[0], train=True)
    save = eng.checkpoint_save

    def fails(format):
        raise torch.OutOfMemoryError("no room")
    a, b = m(xs[0]), m(xs[1])
    eng.checkpoint_save = fails
    with pytest.raises(torch.OutOfMemoryError):
        m(xs[0])
    with pytest.raises(torch.OutOfMemoryError):
        a.backward(dy)
    eng.checkpoint_save = save
    m.zero_grad(set_to_none=True)
    b.backward(dy)
    assert torch.equal(grads(m), exact)
    a.backward(dy)
    assert bool(torch.isfinite(grads(m)).all())


def check_penalty_and_input_gradients(lib, device, manifest, act_dtype, B=2, size=16):
    """A loss over two forwards with the penalty in it, both batches wanting their gradient: the older forward's gradients are those of
    its checkpoint, the newer one's exact, as the plan's own calls give them."""
    from sod100k_amd import _native as N
    xs = [batch(s, device, B, size) for s in (31, 32)]
    dy = K.gradient((B, 1, size, size), torch.float32, 1, device)
    scale = 0.25

    def alone(x, through_checkpoint):
        m = K._net(lib, device, manifest, act_dtype, B)
        m._want_input_grad = True
        m._train_forward_raw(x)
        eng = m.engine_for(x, train=True)
        if through_checkpoint:
            eng.checkpoint_restore(eng.checkpoint_save(N.Q8_INT8), N.Q8_INT8)
        g = m._train_backward_raw(x, dy, scale).clone()
        return torch.cat([g[m._arena.offsets[n]:m._arena.offsets[n] + p.numel()] for n, p in m.named_parameters()]), eng.train_probe(0, "grad0")
    (g0, dx0), (g1, dx1) = alone(xs[0], True), alone(xs[1], False)
    m = net(lib, device, manifest, act_dtype, B=B)
    m.clear_flops()
    leaves = [x.clone().requires_grad_() for x in xs]
    a, b = (m(x) for x in leaves)
    ((a * dy).sum() + (b * dy).sum() + scale * B * m.get_flops()).backward()
    assert torch.equal(leaves[0].grad, dx0) and torch.equal(leaves[1].grad, dx1)
    assert torch.equal(grads(m), g1 + g0)
    assert bool(dx0.abs().sum() > 0) and not torch.equal(g0, g1)


def check_failed_forward(lib, device, manifest):
    """A forward that fails after it has made room (its parameters are packed already): the one that waits still has its checkpoint."""
    xs = [batch(s, device) for s in (31, 32)]
    dy = K.gradient((1, 1, 16, 16), torch.float32, 1, device)
    m = net(lib, device, manifest)
    a, b = m(xs[0]), m(xs[1])
    a.backward(dy)
    want = grads(m)
    del b
    a = m(xs[0])
    eng = m.engine_for(xs[1], train=True)
    forward = eng.forward_train

    def fails(*args, **kwargs):
        raise torch.OutOfMemoryError("no room")
    eng.forward_train = fails
    with pytest.raises(torch.OutOfMemoryError):
        m(xs[1])
    eng.forward_train = forward
    a.backward(dy)
    assert torch.equal(grads(m), want)
    m(xs[1]).backward(dy)                    # and the plan goes on
