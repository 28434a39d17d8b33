"""Further checks of the training operators beside the plan, shared by the emulator suite (tests/test_train_ops_more_emu.py) and the GPU
suite (tests/test_gpu_train_ops_more.py).  Oracles and tolerances: train_ops_cases.py."""
import pytest
import torch

import train_ops_cases as K
from sod100k_amd import _native as N, train_ops as T

# tokens whose channels are all the same number, which a float sum of so many does not give back
CONSTANT = [(shape, dim) for ch in (331, 1000, 2048) for shape, dim in (((3, ch), -1), ((2, ch, 3, 5), 1))] + [((2, 9000), -1)]


def check_constant_tokens(lib, dev, shape, dim, dtype):
    """The mean is that number, the normalised value zero and rstd that of no variance at all: x - m for m near x is exact, so are the
    sums of C equal small multiples of a last place, and their quotient."""
    w, b = K.params(shape[dim], 8, dev)
    for v in (0.1, 1000.1, 30000.7, -3.0e7):
        x = torch.full(shape, v, dtype=torch.float64).to(dtype).to(dev)
        y, mean, rstd, _ = T.layer_norm_forward(lib, x, w, b, dim=dim)
        want = (b if dim == -1 else b.view(1, -1, 1, 1)).expand(shape)
        assert torch.equal(y, want.to(dtype)), v
        assert bool((mean == x.select(dim, 0).float()).all()), v
        assert bool(((rstd.cpu().double() - 1e5 ** 0.5).abs() <= 4 * K.U * 1e5 ** 0.5).all()), v


def check_nan_statistics(lib, dev, shape, dim):
    """A NaN or an infinity in a token leaves no number in its mean and rstd."""
    x = K.activations(shape, torch.float32, 3, dev, rows=dim == -1)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z.select(dim, 1).fill_(bad)
        _, mean, rstd, _ = T.layer_norm_forward(lib, z, dim=dim)
        assert not bool(torch.isfinite(mean).any()) and bool(torch.isnan(rstd).all())


def check_without_gradients(lib, dev, monkeypatch):
    """Under no_grad and inference_mode, parameters or not, the differentiable forms return the same values and keep nothing; where the
    input of a product alone wants a gradient, none of it is kept either."""
    packs = []
    real = T._launch

    def launch(lib, device, what, *args):
        packs.append(what == "csn_q8_pack" or (what == "csn_layer_norm_forward" and args[-1] is not None))
        real(lib, device, what, *args)
    monkeypatch.setattr(T, "_launch", launch)
    g = torch.Generator().manual_seed(1)
    for shape, dim in (((5, 16), -1), ((2, 16, 3, 3), 1)):
        x = torch.randn(shape, generator=g).to(dev)
        w, b = (torch.nn.Parameter(p) for p in K.params(16, 1, dev))
        W = torch.nn.Parameter(torch.randn(8, 16, generator=g).to(dev))
        c = torch.nn.Parameter(torch.randn(8, generator=g).to(dev))
        norm = lambda: T.layer_norm(x, w, b, dim=dim, checkpoint="int8", lib=lib)
        prod = lambda: T.product(x, W, c, dim=dim, lib=lib)
        want = norm().detach(), prod().detach()
        assert any(packs)
        for mode in (torch.no_grad, torch.inference_mode):
            del packs[:]
            with mode():
                got = norm(), prod()
                for call in (lambda: T.layer_norm(x, w, b, dim=dim, checkpoint="fp4", lib=lib), lambda: T.product(x, W, c, dim=dim, checkpoint="fp4", lib=lib)):
                    with pytest.raises(ValueError):
                        call()
                with pytest.raises(TypeError):
                    T.product(x.half(), W, c, dim=dim, lib=lib)
            for p, q in zip(got, want):
                assert torch.equal(p, q) and not p.requires_grad
            assert not any(packs)
        z = x.clone().requires_grad_()
        del packs[:]
        T.product(z, W.detach(), c.detach(), dim=dim, lib=lib).sum().backward()
        assert not any(packs)
        tok = W.detach().sum(0)
        assert torch.allclose(z.grad, (tok if dim == -1 else tok.view(1, -1, 1, 1)).expand(shape), rtol=64 * K.U * 8, atol=64 * K.U * 8)


def check_frozen_norm(lib, dev, monkeypatch):
    """The backward of a norm whose parameters want no gradient asks for none: the same dx, no workspace, no second launch."""
    asked = []
    real = T._launch

    def launch(lib, device, what, *args):
        if what == "csn_layer_norm_backward":
            asked.append([a is not None for a in args[-4:]])      # dweight, dbias, workspace, its size
        real(lib, device, what, *args)
    monkeypatch.setattr(T, "_launch", launch)
    for shape, dim in (((3000, 16), -1), ((2, 16, 30, 30), 1)):
        for ck in (None, "int8"):
            x0, dy = K.activations(shape, torch.float32, 1, dev, rows=dim == -1), K.gradient(shape, torch.float32, 1, dev)
            w, b = K.params(16, 1, dev)
            dx = []
            for train in (True, False):
                del asked[:]
                x = x0.clone().requires_grad_()
                wt, bt = (t.clone().requires_grad_(train) for t in (w, b))
                T.layer_norm(x, wt, bt, dim=dim, checkpoint=ck, lib=lib).backward(dy)
                dx.append(x.grad)
                assert asked == [[train, train, train, True]]
                assert (wt.grad is not None) == train and (bt.grad is not None) == train
            assert torch.equal(*dx)
    _, mean, rstd, _ = T.layer_norm_forward(lib, x0, w, b, dim=1)
    assert T.layer_norm_backward(lib, dy, x0, mean, rstd, w, dim=1, param_grads=False)[1:] == (None, None)


def check_autocast(lib, dev):
    """Inside autocast the product stays in its input's dtype, forward and backward: bit for bit what it is outside."""
    g = torch.Generator().manual_seed(1)
    kind = torch.device(dev).type
    for shape, dim in (((6, 16), -1), ((2, 16, 3, 3), 1)):
        x0, W0, c0 = (torch.randn(s, generator=g).to(dev) for s in (shape, (8, 16), (8,)))
        res = []
        for half in (None, torch.bfloat16, torch.float16):
            x, W, c = (t.clone().requires_grad_() for t in (x0, W0, c0))
            with torch.autocast(kind, dtype=half or torch.bfloat16, enabled=half is not None):
                y = T.product(x, W, c, dim=dim, lib=lib)
                with torch.no_grad():
                    assert torch.equal(T.product(x, W, c, dim=dim, lib=lib), y)
                y.sum().backward()
            assert y.dtype == torch.float32
            res.append((y.detach(), x.grad, W.grad, c.grad))
        for r in res[1:]:
            for p, q in zip(res[0], r):
                assert torch.equal(p, q)
