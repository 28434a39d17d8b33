"""Forwards that wait for their backward (CSNet.set_train_checkpoints) on the CPU emulation of the kernels."""
import pytest
import torch

import waiting_cases as W

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def lib(emu_lanes_lib):
    return emu_lanes_lib[0]


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
def test_emu_refilled_batch(lib, x2_manifest, act_dtype):
    W.check_refilled_batch(lib, CPU, x2_manifest, act_dtype)


def test_uses_of_the_workspace_wait_for_each_other(lib, x2_manifest, monkeypatch):
    """Every launch of a training plan on another stream than the one before waits for an event behind that one (the emulator runs the
    launches, stand-ins for streams and events write down what is asked of them)."""
    log = []

    class Stream:
        def __init__(self, n):
            self.cuda_stream = n

        def wait_event(self, e):
            log.append(("wait", self.cuda_stream, e.recorded))

    class Event:
        recorded = None

        def record(self, s):
            self.recorded = s.cuda_stream
            log.append(("record", s.cuda_stream))

    class Device:
        type = "cuda"

    m = W.net(lib, CPU, x2_manifest)
    x = W.batch(31, CPU)
    y, _ = m._train_forward_raw(x)
    eng = m.engine_for(x, train=True)
    dy = torch.ones_like(y)
    flat = torch.zeros(m._arena.n_param_floats)
    now = [Stream(1)]
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    real = eng.device
    uses = [lambda: eng.refresh(m._arena.flat), lambda: eng.forward_train(x, m._arena.flat, m._flop_tab, torch.zeros(1, dtype=torch.float64)),
            lambda: held.append(save()), lambda: eng.checkpoint_restore(held[-1], 0),
            lambda: eng.backward(x, dy, m._arena.flat, flat, m._flop_tab, 0.0), lambda: eng.train_probe(1, "z")]
    held = []

    def save():
        empty = torch.empty
        with monkeypatch.context() as p:      # (the buffer itself lies on the host)
            p.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
            return eng.checkpoint_save(0)
    eng.device = Device()
    try:
        uses[0]()
        uses[1]()
        assert log == [("record", 1)] * 2                     # one stream: nothing to wait for
        for n, use in enumerate(uses, 2):
            del log[:]
            now[0] = Stream(n)
            use()
            assert log == [("wait", n, n - 1), ("record", n)]
        del log[:]
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        now[0] = Stream(99)
        uses[0]()
        assert log == []                                      # inside a capture the order is the caller's
    finally:
        eng.device = real


def test_emu_changed_parameters(lib, x2_manifest):
    W.check_changed_parameters(lib, CPU, x2_manifest)


def test_emu_failed_save(lib, x2_manifest):
    W.check_failed_save(lib, CPU, x2_manifest)


def test_emu_penalty_and_input_gradients(lib, x2_manifest):
    W.check_penalty_and_input_gradients(lib, CPU, x2_manifest, "fp32")


def test_emu_failed_forward(lib, x2_manifest):
    W.check_failed_forward(lib, CPU, x2_manifest)
