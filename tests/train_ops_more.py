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


# ---- more tokens than a launch has blocks: the loops of the register forms -------------------------------------------------------
# Every form of csrc/k_norm.hip with blocks that take a second token or tile: rows by lanes per token (8, 16, 32, 64, 256, 1024) and
# pieces per lane (1, 2), maps by threads, lanes across the pixels and channels per lane, in whole cache lines and not (runs).
MANY_ROWS = [(100000, 40), (50000, 100), (25000, 200), (9000, 512), (7000, 1000), (5000, 2048), (2600, 3000), (1300, 5000), (700, 12000)]
MANY_MAPS = [(36, 40, 88, 88), (70, 128, 57, 57), (36, 200, 64, 64), (40, 300, 44, 44), (20, 700, 44, 44), (10, 1100, 44, 44), (10, 2048, 28, 28)]


def _per_token(t, dim):
    """[channels, tokens] in 64 bits, where the tensor lies."""
    t = t.detach().double()
    return t.reshape(-1, t.shape[-1]).t() if dim == -1 else t.movedim(1, 0).reshape(t.shape[1], -1)


def check_many_tokens(lib, dev, shape, dim, dtype):
    """Forward and backward of random tokens against the formulas in 64 bits, from the tensor and from both checkpoints.  Tolerances:
    train_ops_cases.py."""
    rows = dim == -1
    x, dy = K.activations(shape, dtype, 1, "cpu", rows=rows).to(dev), K.gradient(shape, dtype, 1, "cpu").to(dev)
    w, b = K.params(shape[dim], 1, dev)
    wd, bd = w.double()[:, None], b.double()[:, None]
    ch = shape[dim]
    y, mean, rstd, _ = T.layer_norm_forward(lib, x, w, b, dim=dim)
    t = _per_token(x, dim)
    m = t.sum(0) / ch
    d = t - m
    r = 1 / torch.sqrt((d * d).sum(0) / ch + 1e-5)
    k, half = 64 * K.U, K.HALF[dtype]
    dm = k * t.abs().amax(0)
    dr = k + (dm * r) ** 2
    assert bool(((mean.double().reshape(-1) - m).abs() <= dm).all())
    assert bool(((rstd.double().reshape(-1) - r).abs() <= dr * r).all())
    want = d * r * wd + bd
    tol = wd * (dm * r + d.abs() * r * dr) + k * (bd.abs() + want.abs()) + half * want.abs()
    assert bool(((_per_token(y, dim) - want).abs() <= tol).all())
    del want, tol, d, t
    m, r = mean.double().reshape(-1), rstd.double().reshape(-1)
    g0 = _per_token(dy, dim)
    g = g0 * wd
    for fmt in (None,) + K.FORMATS:
        src = x
        if fmt is not None:
            y2, m2, r2, src = T.layer_norm_forward(lib, x, w, b, dim=dim, checkpoint=fmt)
            assert torch.equal(y, y2) and torch.equal(mean, m2) and torch.equal(rstd, r2)
            del y2
            p = T.q8_pack(lib, x, fmt, start_dim=-1 if rows else 2)
            assert torch.equal(p.codes, src.codes) and torch.equal(p.scales, src.scales)
        dx, dw, db = T.layer_norm_backward(lib, dy, src, mean, rstd, w, dim=dim)
        xh = (_per_token(x if fmt is None else T.q8_unpack(lib, src), dim) - m) * r
        gx = g * xh
        want = r * (g - g.sum(0) / ch - xh * (gx.sum(0) / ch))
        tol = k * r * (g.abs() + g.abs().sum(0) / ch + xh.abs() * (gx.abs().sum(0) / ch)) + half * want.abs()
        assert bool(((_per_token(dx, dim) - want).abs() <= tol).all())
        gx = g0 * xh
        assert bool(((dw.double() - gx.sum(1)).abs() <= 1024 * K.U * gx.abs().sum(1)).all())
        assert bool(((db.double() - g0.sum(1)).abs() <= 1024 * K.U * g0.abs().sum(1)).all())


def check_refusals_of_workspaces(lib):
    """Descriptors that need a workspace, and calls that bring none, too little or a misaligned one (host code only: no pointer is
    followed)."""
    import ctypes as C
    p, big = C.c_void_p(4096), 1 << 40
    for d in (N.NormDesc(N.LAYOUT_ROWS, N.DTYPE_F32, 100000, 8, 1, 1e-5, 0), N.NormDesc(N.LAYOUT_PLANAR, N.DTYPE_BF16, 4, 40, 3000, 1e-5, 0)):
        need = lib.csn_layer_norm_workspace_bytes(C.byref(d))
        assert need > 0
        so, sc = (8, 0) if d.layout == N.LAYOUT_ROWS else (120000, 3000)
        for ws, n in ((p, need - 1), (None, big), (C.c_void_p(4098), big), (p, 0)):
            for dw, db in ((p, p), (None, p), (p, None)):
                st = lib.csn_layer_norm_backward(C.byref(d), p, so, sc, p, so, sc, None, None, p, p, None, p, dw, db, ws, n, None)
                assert st == 1 and b"workspace" in lib.csn_last_hip_error()
    for d in (N.ProductDesc(N.LAYOUT_ROWS, N.DTYPE_F32, 0, 0, 100000, 1, 8, 8), N.ProductDesc(N.LAYOUT_PLANAR, N.DTYPE_BF16, 1, 0, 4, 3000, 40, 70)):
        need = lib.csn_product_weight_grad_workspace_bytes(C.byref(d))
        assert need > 0
        for ws, n in ((p, need - 1), (None, big), (C.c_void_p(4098), big), (p, 0)):
            st = lib.csn_product_weight_grad(C.byref(d), p, 210000, 3000, p, p, p, p, ws, n, None)
            assert st == 1 and b"workspace" in lib.csn_last_hip_error()


def check_outputs_end_where_they_end(lib, dev):
    """Memory behind the gradients and the workspaces of calls with several slabs stays as it was."""
    import ctypes as C
    stream = torch.cuda.current_stream().cuda_stream if torch.device(dev).type == "cuda" else None

    def buf(n, t=torch.float32):
        return torch.full((n + 64,), 77, dtype=t, device=dev)
    for dtype, dt in ((torch.float32, 0), (torch.bfloat16, 1)):
        for rows, o, cin, cout, p in ((True, 2000, 33, 70, 1), (True, 700, 8, 3, 1), (False, 3, 37, 21, 301), (False, 2, 130, 5, 700)):
            xs = (o, cin) if rows else (o, cin, p)
            x, dy = K.activations(xs, dtype, 1, dev, rows=rows), K.gradient((o, cout) if rows else (o, cout, p), dtype, 1, dev)
            for fmt, f in (("int8", 0), ("e4m3", 1)):
                q = T.q8_pack(lib, x, fmt, start_dim=-1 if rows else 2)
                d = N.ProductDesc(int(rows), dt, f, 0, o, p, cin, cout)
                need = lib.csn_product_weight_grad_workspace_bytes(C.byref(d))
                assert need > 0
                dw, db, ws = buf(cin * cout), buf(cout), buf(need, torch.uint8)
                N.check(lib, lib.csn_product_weight_grad(C.byref(d), dy.data_ptr(), cout if rows else cout * p, 0 if rows else p, q.codes.data_ptr(),
                                                         q.scales.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, stream), "product")
                w2, b2 = T.product_weight_grad(lib, dy, q, dim=-1 if rows else 1)
                assert torch.equal(dw[:-64], w2.reshape(-1)) and torch.equal(db[:-64], b2)
                for t in (dw, db, ws):
                    assert bool((t[-64:] == 77).all())
        for rows, o, c, p in ((True, 4000, 33, 1), (True, 40, 2100, 1), (False, 3, 7, 1301), (False, 2, 300, 333)):
            shape = (o, c) if rows else (o, c, p)
            x, dy = K.activations(shape, dtype, 1, dev, rows=rows), K.gradient(shape, dtype, 1, dev)
            _, mean, rstd, _ = T.layer_norm_forward(lib, x, dim=-1 if rows else 1)
            d = N.NormDesc(int(rows), dt, o, c, p, 1e-5, 0)
            need = lib.csn_layer_norm_workspace_bytes(C.byref(d))
            assert need > 0
            dx, dw, db, ws = buf(x.numel(), dtype), buf(c), buf(c), buf(need, torch.uint8)
            so, sc = (c, 0) if rows else (c * p, p)
            N.check(lib, lib.csn_layer_norm_backward(C.byref(d), dy.data_ptr(), so, sc, x.data_ptr(), so, sc, None, None, mean.data_ptr(), rstd.data_ptr(),
                                                     None, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, stream), "norm")
            ref = T.layer_norm_backward(lib, dy, x, mean, rstd, dim=-1 if rows else 1)
            for t, r in zip((dx, dw, db), ref):
                assert torch.equal(t[:-64], r.reshape(-1))
            for t in (dx, dw, db, ws):
                assert bool((t[-64:] == 77).all())
