"""Checks of the training operators beside the plan (layer norm, 8-bit checkpoints, product gradients), shared by the emulator
suite (tests/test_train_ops_emu.py, host tensors) and the GPU suite (tests/test_gpu_train_ops.py).  Oracles are 64-bit torch code on
the host, written from the definitions in include/csnet_hip.h.

Tolerances.  u = 2^-24 is the largest relative error of one float operation; a stored bfloat16 is off by at most 2^-9 + its
double-rounding share, counted as 2^-8 of the value.  Every reduction of the kernels adds at most CHAIN numbers one after another in
float before it goes to a tree or to double, so a sum is off by at most CHAIN u sum|terms|; the handful of operations around a sum
are covered by taking CHAIN = 64 for the sums over channels (normalised values: 64 u of the largest magnitude involved) and
CHAIN = 1024 for the sums over tokens."""
import ctypes as C
import math

import pytest
import torch

from sod100k_amd import _native as N, train_ops as T

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
FORMATS = ("int8", "e4m3")
DTYPES = (torch.float32, torch.bfloat16)


# ---- oracles --------------------------------------------------------------------------------------------------------------
def _grid(fmt):
    """All finite values of the code grid, ascending, in 64 bits, and their codes."""
    if fmt == "int8":
        vals = [(float(v), v & 255) for v in range(-127, 128)]
    else:
        vals = []
        for c in range(256):
            s, e, m = c >> 7, (c >> 3) & 15, c & 7
            if (e, m) == (15, 7):
                continue
            vals.append(((-1.0) ** s * ((8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9), c))
    vals.sort()
    return vals


def oracle_pack(x, fmt, start):
    """(values, exponents) by the definition: the smallest power of two that keeps the block's largest value in range, then the
    nearest number of the grid, ties to the even code."""
    x = x.detach().cpu().double()
    rows = x.flatten(start) if start != -1 else x
    lead, cols = rows.shape[:-1], rows.shape[-1]
    rows = rows.reshape(-1, cols)
    top = 127.0 if fmt == "int8" else 448.0
    edge = 127.5 if fmt == "int8" else 464.0        # from here (int8) / beyond here (e4m3) a value would round out of range
    grid = _grid(fmt)
    limit = edge * 2.0 ** (121 if fmt == "int8" else 119)      # (rounds to 2^128: kept as NaN like the infinities)
    g = torch.tensor([v for v, _ in grid], dtype=torch.float64)
    even = torch.tensor([(c & 1) == 0 for _, c in grid])
    nb = -(-cols // 32)
    vals, exps = torch.empty_like(rows), torch.empty(rows.shape[0], nb, dtype=torch.int64)
    for b in range(nb):
        blk = rows[:, 32 * b:32 * b + 32]
        fin = (blk.abs() < limit) if fmt == "int8" else (blk.abs() <= limit)
        amax = torch.where(fin, blk.abs(), 0.0).amax(1)
        for r in range(rows.shape[0]):
            e = -95
            a = float(amax[r])
            if a > 0:
                e = max(e, math.frexp(a)[1] - 12)
                while (a * 2.0 ** -e >= edge) if fmt == "int8" else (a * 2.0 ** -e > edge):
                    e += 1
            exps[r, b] = e + 127
        s = torch.exp2((exps[:, b] - 127).double())[:, None]
        t = torch.where(fin, blk, 0.0) / s
        hi = torch.searchsorted(g, t.contiguous()).clamp(max=len(g) - 1)
        lo = (hi - 1).clamp(min=0)
        dl, dh = (t - g[lo]).abs(), (g[hi] - t).abs()
        pick = torch.where((dh < dl) | ((dh == dl) & even[hi]), hi, lo)
        v = g[pick] * s
        vals[:, 32 * b:32 * b + 32] = torch.where(fin, v, torch.full_like(v, float("nan")))
        assert float((t.abs().amax() if t.numel() else torch.zeros(()))) < top * 1.04
    return vals.reshape(x.shape), exps.reshape(lead + (nb,)).to(torch.uint8)


def _tok(x, rows):
    """[channels, tokens] in 64 bits."""
    x = x.detach().cpu().double()
    return x.reshape(-1, x.shape[-1]).t() if rows else x.movedim(1, 0).reshape(x.shape[1], -1)


def _untok(t, like, rows):
    if rows:
        return t.t().reshape(like.shape)
    return t.reshape((like.shape[1], like.shape[0]) + tuple(like.shape[2:])).movedim(0, 1)


def same(a, b):
    """Equal, NaN where NaN."""
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def activations(shape, dtype, seed, dev="cpu", rows=True):
    g = torch.Generator().manual_seed(seed)
    ch = shape[-1] if rows else shape[1]
    spread, off = torch.exp(0.5 * torch.randn(ch, generator=g)), 0.5 * torch.randn(ch, generator=g)
    v = (1, -1) + (1,) * (len(shape) - 2)
    x = torch.randn(shape, generator=g)
    x = x * spread + off if rows else x * spread.view(v) + off.view(v)
    return x.to(dtype).to(dev)


def gradient(shape, dtype, seed, dev="cpu"):
    return (1e-2 * torch.randn(shape, generator=torch.Generator().manual_seed(seed + 1000))).to(dtype).to(dev)


def params(ch, seed, dev="cpu"):
    g = torch.Generator().manual_seed(seed + 2000)
    return (1 + 0.2 * torch.randn(ch, generator=g)).to(dev), (0.2 * torch.randn(ch, generator=g)).to(dev)


# ---- checks ---------------------------------------------------------------------------------------------------------------
def check_pack(lib, x, fmt, start):
    q = T.q8_pack(lib, x, fmt, start_dim=start)
    v, e = oracle_pack(x, fmt, start)
    assert torch.equal(q.scales.cpu(), e)
    for dt in DTYPES:        # both output types hold the values exactly
        assert same(T.q8_unpack(lib, q, dt).cpu().double(), v)
    code = q.codes.cpu()[torch.isnan(v)]
    assert bool((code == (128 if fmt == "int8" else 127)).all())
    return q


def block_edge_values(dtype):
    """Rows of 32 whose largest value sits on both sides of where the exponent changes, at the ends of the type's range and with
    nothing, zeros, infinities and NaN."""
    tiny = 2.0 ** -126
    big = float(torch.finfo(dtype).max)
    tops = [127.0, 127.5, 127.4375, 127.75, 128.0, 448.0, 464.0, 463.0, 466.0, 480.0, 1.9921875, 1.8125, 1.0, 2.0 ** -94, 2.0 ** -95, 2.0 ** -96,
            tiny, 2.0 ** -133, big, big / 2, 0.0]
    rows = []
    for i, t in enumerate(tops):
        r = torch.linspace(-1, 1, 32, dtype=torch.float64) * t * 0.99
        r[(7 * i) % 32] = t if i % 2 else -t
        rows.append(r)
    x = torch.stack(rows).to(torch.float32).clamp(-big, big)
    bad = torch.randn(5, 32, generator=torch.Generator().manual_seed(3))
    bad[0, 3], bad[1, 0], bad[2, 31] = float("inf"), float("-inf"), float("nan")
    bad[3, :] = float("nan")
    bad[4, ::2] = float("inf")
    return torch.cat([x, bad]).to(dtype)


def every_code_once(fmt, dev="cpu"):
    """All 256 codes in blocks whose exponents differ: what unpack returns, and what packing that again gives."""
    codes = torch.arange(256, dtype=torch.int64).repeat(3).to(torch.uint8).view(3, 256)
    scales = torch.tensor([127, 32, 200], dtype=torch.uint8).view(3, 1).repeat(1, 8).contiguous()
    val = dict((c, v) for v, c in _grid(fmt))
    want = torch.tensor([val.get(c, float("nan")) for c in range(256)], dtype=torch.float64).repeat(3, 1)
    want = want * torch.exp2(scales[:, :1].double() - 127)
    return T.Q8(codes.to(dev), scales.to(dev), fmt, -1), want


def check_norm_forward(lib, x, w, b, dim, checkpoint=None, eps=1e-5):
    rows = dim == -1
    y, mean, rstd, q = T.layer_norm_forward(lib, x, w, b, dim=dim, eps=eps, checkpoint=checkpoint)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    t = _tok(x, rows)
    ch = t.shape[0]
    m = t.sum(0) / ch
    var = ((t - m) ** 2).sum(0) / ch
    r = 1 / torch.sqrt(var + eps)
    wd = torch.ones(ch, 1, dtype=torch.float64) if w is None else w.cpu().double()[:, None]
    bd = torch.zeros(ch, 1, dtype=torch.float64) if b is None else b.cpu().double()[:, None]
    want = (t - m) * r * wd + bd
    biggest = t.abs().amax(0) if ch else t.new_zeros(t.shape[1])
    k = 64 * U
    # the mean is off by k max|x|; the variance by k of itself plus the square of that; both move y
    dm = k * biggest
    dr = k + (dm * r) ** 2
    assert bool(((mean.cpu().double().reshape(-1) - m).abs() <= dm).all())
    assert bool(((rstd.cpu().double().reshape(-1) - r).abs() <= dr * r).all())
    tol = wd.abs() * (dm * r + (t - m).abs() * r * dr) + k * (bd.abs() + want.abs()) + HALF[x.dtype] * want.abs()
    err = (_tok(y, rows) - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())
    if checkpoint:
        v, e = oracle_pack(x, checkpoint, -1 if rows else 2)
        assert torch.equal(q.scales.cpu(), e) and same(T.q8_unpack(lib, q).cpu().double(), v)
    else:
        assert q is None
    return y, mean, rstd, q


def check_norm_backward(lib, dy, x, mean, rstd, w, dim, q=None):
    rows = dim == -1
    dx, dw, db = T.layer_norm_backward(lib, dy, x if q is None else q, mean, rstd, w, dim=dim)
    t = _tok(x, rows) if q is None else _tok(oracle_pack(x, q.format, q.start_dim)[0], rows)
    g0, ch = _tok(dy, rows), t.shape[0]
    m, r = mean.cpu().double().reshape(-1), rstd.cpu().double().reshape(-1)
    wd = torch.ones(ch, 1, dtype=torch.float64) if w is None else w.cpu().double()[:, None]
    xh, g = (t - m) * r, g0 * wd
    c1, c2 = g.sum(0) / ch, (g * xh).sum(0) / ch
    want = r * (g - c1 - xh * c2)
    a1, a2 = g.abs().sum(0) / ch, (g * xh).abs().sum(0) / ch
    k = 64 * U
    tol = k * r * (g.abs() + a1 + xh.abs() * a2) + HALF[dy.dtype] * want.abs()
    assert dx.dtype == dy.dtype and dx.shape == dy.shape
    err = (_tok(dx, rows) - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())
    k = 1024 * U
    assert bool(((dw.cpu().double() - (g0 * xh).sum(1)).abs() <= k * (g0 * xh).abs().sum(1)).all())
    assert bool(((db.cpu().double() - g0.sum(1)).abs() <= k * g0.abs().sum(1)).all())
    return dx, dw, db


def check_product(lib, dy, x, fmt, dim):
    rows = dim == -1
    q = T.q8_pack(lib, x, fmt, start_dim=-1 if rows else 2)
    dw, db = T.product_weight_grad(lib, dy, q, dim=dim)
    v = _tok(oracle_pack(x, fmt, q.start_dim)[0], rows)
    g = _tok(dy, rows)
    k = 1024 * U
    err, tol = (dw.cpu().double() - g @ v.t()).abs(), k * (g.abs() @ v.abs().t())
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())
    assert bool(((db.cpu().double() - g.sum(1)).abs() <= k * g.abs().sum(1)).all())
    return dw, db


# shapes: (shape, dim) -- one token, one channel, odd widths, a short last block, rows wider than a block's registers, planes that end
# inside a block and a vector
NORM_SHAPES = [((1, 1), -1), ((1, 2048), -1), ((7, 8), -1), ((5, 33), -1), ((130, 64), -1), ((3, 331), -1), ((2, 9, 80), -1), ((2, 5000), -1),
               ((1, 20000), -1), ((70, 1000), -1), ((1, 1, 1, 1), 1), ((2, 79, 5, 7), 1), ((1, 40, 28, 28), 1), ((3, 20, 1, 1), 1),
               ((2, 8, 33), 1), ((1, 300, 6, 6), 1), ((2, 64, 16, 16), 1), ((1, 2, 100, 3), 1), ((1, 1100, 4, 8), 1), ((1, 64, 40, 40), 1), ((1, 3000, 5, 7), 1), ((1, 5000, 1, 3), 1), ((1, 33000), -1),
               ((1, 150, 6, 6), 1), ((1, 600, 5, 5), 1)]
PACK_SHAPES = [((1,), -1), ((3, 31), -1), ((2, 32), -1), ((5, 33), -1), ((4, 64), -1), ((3, 7, 100), -1), ((2, 3, 5, 9), 2), ((1, 4, 8, 8), 2),
               ((2, 2, 1, 1), 2), ((3, 40, 14, 14), 2)]
# (outer dims of x, cin, cout, dim)
PRODUCT_SHAPES = [((1,), 1, 1, -1), ((7,), 8, 3, -1), ((65,), 33, 70, -1), ((300,), 64, 48, -1), ((2, 50), 130, 17, -1), ((1, 1, 1), 1, 1, 1), ((2, 3, 3), 37, 21, 1),
                  ((3, 8, 8), 16, 64, 1), ((1, 13, 17), 40, 33, 1), ((2, 16, 20), 130, 20, 1), ((5, 12, 12), 18, 13, 1)]


def product_tensors(dims, cin, cout, dim, dtype, seed, dev="cpu"):
    mk = (lambda c: tuple(dims) + (c,)) if dim == -1 else (lambda c: (dims[0], c) + tuple(dims[1:]))
    return (activations(mk(cin), dtype, seed, dev, rows=dim == -1), gradient(mk(cout), dtype, seed, dev))


def check_slices(lib, dev, dtype):
    """Inputs that are slices of wider tensors, broadcast gradients and permuted tensors give what their dense copies give."""
    wide = activations((6, 50), dtype, 5, dev)
    dyw = gradient((6, 50), dtype, 5, dev)
    w, b = params(37, 5, dev)
    for x, dy in ((wide[:, 5:42], dyw[:, 9:46]), (wide[:, 8:45], dyw[:1, 3:40].expand(6, 37)), (wide[::2, 1:38], dyw[1:4, 1:38]),
                  (wide.t()[:37].t(), dyw.t()[2:39].t())):
        run = lambda x, dy: _all_of(T, lib, x, dy, w, b, -1)
        for s, d in zip(run(x, dy), run(x.clone().contiguous(), dy.clone().contiguous())):
            assert torch.equal(s, d)
    wide = activations((3, 20, 6, 10), dtype, 6, dev, rows=False)
    dyw = gradient((3, 20, 6, 10), dtype, 6, dev)
    w, b = params(11, 6, dev)
    for x, dy in ((wide[:, 4:15], dyw[:, 9:20]), (wide[1:, 4:15], dyw[:1, 9:20].expand(2, 11, 6, 10)),
                  (wide[:, 4:15, 1:5, ::2], dyw[:, 9:20, 2:, :5]), (wide[:, 1:12].to(memory_format=torch.channels_last), dyw[:, :11])):
        run = lambda x, dy: _all_of(T, lib, x, dy, w, b, 1)
        for s, d in zip(run(x, dy), run(x.clone(memory_format=torch.contiguous_format).contiguous(), dy.clone().contiguous())):
            assert torch.equal(s, d)


def _all_of(T, lib, x, dy, w, b, dim):
    out = []
    for fmt in (None,) + FORMATS:
        y, mean, rstd, q = T.layer_norm_forward(lib, x, w, b, dim=dim, checkpoint=fmt)
        out += [y, mean, rstd] + ([] if q is None else [q.codes, q.scales])
        out += T.layer_norm_backward(lib, dy, x if q is None else q, mean, rstd, w, dim=dim)
        if q is not None:
            out += T.product_weight_grad(lib, dy, q, dim=dim)
            p = T.q8_pack(lib, x, fmt, start_dim=-1 if dim == -1 else 2)
            out += [p.codes, p.scales]
    return out


def check_empty(lib, dev):
    for shape, dim in (((0, 5), -1), ((0, 5, 3, 3), 1), ((2, 5, 0, 3), 1)):
        x = torch.empty(shape, device=dev)
        y, mean, rstd, q = T.layer_norm_forward(lib, x, dim=dim, checkpoint="int8")
        assert y.shape == x.shape and mean.numel() == 0 and T.q8_unpack(lib, q).shape == x.shape
        for src in (x, q):
            dx, dw, db = T.layer_norm_backward(lib, x, src, mean, rstd, dim=dim)
            assert dx.shape == x.shape and not dw.any() and not db.any()
        dw, db = T.product_weight_grad(lib, torch.empty(shape, device=dev), q, dim=dim)
        assert dw.shape == (5, 5) and not dw.any() and not db.any()


def check_bad_tokens_stay_alone(lib, dev, dtype):
    """A token with an infinity or a NaN is lost; the others' results are bit for bit what they are without it."""
    for shape, dim in (((9, 40), -1), ((2, 40, 5, 9), 1)):
        rows = dim == -1
        x, dy = activations(shape, dtype, 7, dev, rows=rows), gradient(shape, dtype, 7, dev)
        w, b = params(40, 7, dev)
        bad = x.clone()
        sel = [(2, 3), (5, 39)] if rows else [(0, 3, 0, 0), (1, 39, 4, 8)]
        bad[sel[0]], bad[sel[1]] = float("nan"), float("inf")
        y0, m0, r0, _ = T.layer_norm_forward(lib, x, w, b, dim=dim)
        y1, m1, r1, _ = T.layer_norm_forward(lib, bad, w, b, dim=dim)
        d0, d1 = (T.layer_norm_backward(lib, dy, xx, mm, rr, w, dim=dim)[0] for xx, mm, rr in ((x, m0, r0), (bad, m1, r1)))
        lost = torch.zeros(m0.shape, dtype=torch.bool)
        for s in sel:
            lost[s[:1] if rows else s[:1] + s[2:]] = True
        keep = ~lost
        for p, q in ((y0, y1), (d0, d1)):
            p, q = (t.cpu() if rows else t.cpu().movedim(1, -1) for t in (p, q))
            assert torch.equal(p[keep], q[keep]) and torch.isnan(q[lost]).all()


def check_constant_and_far(lib, dev):
    """Tokens without variance normalise to the bias; a mean far beyond the spread costs digits of x, not of the statistics."""
    for shape, dim in (((4, 100), -1), ((2, 100, 3, 5), 1)):
        x = torch.full(shape, 3.0, device=dev)
        w, b = params(100, 8, dev)
        y, mean, rstd, _ = T.layer_norm_forward(lib, x, w, b, dim=dim)
        want = b if dim == -1 else b.view(1, -1, 1, 1)
        assert torch.equal(y, want.expand(shape)) and bool((mean == 3).all())
        assert bool(((rstd.cpu().double() - 1e5 ** 0.5).abs() <= 4 * U * 1e5 ** 0.5).all())
        check_norm_forward(lib, activations(shape, torch.float32, 9, dev, rows=dim == -1) + 1000.0, w, b, dim)


def check_determinism(lib, dev):
    x, dy = activations((3, 70, 9, 31), torch.bfloat16, 10, dev, rows=False), gradient((3, 70, 9, 31), torch.bfloat16, 10, dev)
    w, b = params(70, 10, dev)
    first = _all_of(T, lib, x, dy, w, b, 1)
    for _ in range(2):
        for p, q in zip(first, _all_of(T, lib, x, dy, w, b, 1)):
            assert torch.equal(p, q)


def check_against_differences(lib, dev):
    """Gradients of the differentiable forms against central differences of their own forwards, in float.  With steps of h = 2^-6 in
    numbers of size 1 a difference quotient of F = sum(y r) is off by about u sqrt(n) |F'| / h (rounding) and h^2 |F'''| / 6, both
    well below 1 % of a directional derivative along a random direction."""
    for shape, dim in (((6, 24), -1), ((2, 24, 3, 3), 1)):
        rows = dim == -1
        x = activations(shape, torch.float32, 11, dev, rows=rows)
        w, b = params(24, 11, dev)
        r = torch.randn(shape, generator=torch.Generator().manual_seed(12)).to(dev)
        f = lambda *a: float((T.layer_norm(a[0], a[1], a[2], dim=dim, lib=lib).double() * r.double()).sum())
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        (T.layer_norm(*leaves, dim=dim, lib=lib) * r).sum().backward()
        for i, leaf in enumerate(leaves):
            v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(13 + i)).to(dev)
            v = v + leaf.grad / leaf.grad.norm() * v.norm()         # (not nearly perpendicular to the gradient)
            h = 2.0 ** -6 / float(v.abs().max())
            args = [t.detach() for t in leaves]
            up, dn = list(args), list(args)
            up[i], dn[i] = args[i] + h * v, args[i] - h * v
            num, ana = (f(*up) - f(*dn)) / (2 * h), float((leaf.grad.double() * v.double()).sum())
            assert abs(num - ana) <= 1e-2 * abs(ana), (shape, i, num, ana)


def check_block_of_operators(lib, dev, dtype):
    """Norm and product as a block uses them, with and without 8-bit checkpoints: the outputs do not depend on how the inputs are
    kept, the gradients are those of the values that were kept."""
    for shape, dim, start in (((40, 48), -1, -1), ((2, 48, 5, 7), 1, 2)):
        rows = dim == -1
        x0 = activations(shape, dtype, 14, dev, rows=rows)
        w, b = params(48, 14, dev)
        g = torch.Generator().manual_seed(15)
        W, c = (0.15 * torch.randn(32, 48, generator=g)).to(dev), (0.1 * torch.randn(32, generator=g)).to(dev)
        outs = {}
        for ck in (None, "int8", "e4m3"):
            leaves = [t.clone().requires_grad_() for t in (x0, w, b, W, c)]
            h = T.layer_norm(leaves[0], leaves[1], leaves[2], dim=dim, checkpoint=ck, lib=lib)
            y = T.product(h, leaves[3], leaves[4], dim=dim, checkpoint=ck or "int8", lib=lib)
            dy = gradient(y.shape, dtype, 16, dev)
            y.backward(dy)
            outs[ck] = (y.detach(), h.detach(), [t.grad for t in leaves])
        for ck in ("int8", "e4m3"):
            y, h, grads = outs[ck]
            assert torch.equal(y, outs[None][0]) and torch.equal(h, outs[None][1])
            g0, v = _tok(dy, rows), _tok(oracle_pack(h, ck, start)[0], rows)
            assert bool(((grads[3].cpu().double() - g0 @ v.t()).abs() <= 1024 * U * (g0.abs() @ v.abs().t())).all())
            assert bool(((grads[4].cpu().double() - g0.sum(1)).abs() <= 1024 * U * g0.abs().sum(1)).all())
            # through the norm: its own backward on the checkpoint's values, from the library product's input gradient
            wt = W.cpu().double().to(dtype).double()
            dh = T._product(dy, W.t().contiguous(), None, rows)
            q = T.q8_pack(lib, x0, ck, start_dim=start)
            _, mean, rstd, _ = T.layer_norm_forward(lib, x0, w, b, dim=dim)
            dx, dw, db = check_norm_backward(lib, dh, x0, mean, rstd, w, dim, q=q)
            assert torch.equal(dx, grads[0]) and torch.equal(dw, grads[1]) and torch.equal(db, grads[2])
            del wt


def check_refusals(lib, dev):
    """Calls that the documentation does not allow raise before anything is launched."""
    import pytest
    x = torch.zeros(4, 8, device=dev)
    m = torch.zeros(2, 8, 3, 3, device=dev)
    q = T.q8_pack(lib, x)
    _, mean, rstd, _ = T.layer_norm_forward(lib, x)
    for exc, call in (
            (ValueError, lambda: T.q8_pack(lib, x, "int4")), (TypeError, lambda: T.q8_pack(lib, x.half())),
            (ValueError, lambda: T.q8_pack(lib, x, start_dim=1)), (ValueError, lambda: T.q8_pack(lib, x, start_dim=2)),
            (TypeError, lambda: T.q8_unpack(lib, q, torch.float16)),
            (ValueError, lambda: T.q8_unpack(lib, q._replace(scales=q.scales[:3]))),
            (TypeError, lambda: T.q8_unpack(lib, q._replace(codes=q.codes.float()))),
            (ValueError, lambda: T.q8_unpack(lib, q._replace(codes=q.codes[:, ::2]))),
            (ValueError, lambda: T.layer_norm_forward(lib, m, dim=2)), (ValueError, lambda: T.layer_norm_forward(lib, m, dim=7)),
            (TypeError, lambda: T.layer_norm_forward(lib, x.double())),
            (ValueError, lambda: T.layer_norm_forward(lib, x, torch.ones(7, device=dev))),
            (TypeError, lambda: T.layer_norm_forward(lib, x, torch.ones(8, device=dev, dtype=torch.bfloat16))),
            (RuntimeError, lambda: T.layer_norm_forward(lib, x, eps=0.0)), (RuntimeError, lambda: T.layer_norm_forward(lib, x, eps=-1.0)),
            (RuntimeError, lambda: T.layer_norm_forward(lib, x, eps=float("nan"))),
            (RuntimeError, lambda: T.layer_norm_forward(lib, torch.zeros(4, 0, device=dev))),
            (ValueError, lambda: T.layer_norm_backward(lib, x, x[:3], mean, rstd)),
            (TypeError, lambda: T.layer_norm_backward(lib, x, x.bfloat16(), mean, rstd)),
            (ValueError, lambda: T.layer_norm_backward(lib, x, x, mean[:3], rstd)),
            (ValueError, lambda: T.layer_norm_backward(lib, x, x, mean, rstd.double())),
            (ValueError, lambda: T.layer_norm_backward(lib, m, T.q8_pack(lib, m), m[:, 0], m[:, 0], dim=1)),
            (ValueError, lambda: T.product_weight_grad(lib, x[:3], q)), (ValueError, lambda: T.product_weight_grad(lib, m, q, dim=1)),
            (TypeError, lambda: T.product_weight_grad(lib, x.half(), q)),
            (ValueError, lambda: T.product(x, torch.zeros(3, 7, device=dev), lib=lib)),
            (ValueError, lambda: T.product(x, torch.zeros(3, 8, device=dev), checkpoint="fp4", lib=lib))):
        with pytest.raises(exc):
            call()


def check_refusals_of_the_abi(lib):
    """The C entry points return CSN_E_INVALID and name the reason; no pointer is followed (host code only)."""
    def bad(status, word):
        assert status == 1 and word in lib.csn_last_hip_error().decode(), lib.csn_last_hip_error()
    p = C.c_void_p(4096)      # never followed
    bad(lib.csn_q8_pack(p, 7, 1, 1, 1, 1, 1, 0, p, p, None), "dtype")
    bad(lib.csn_q8_pack(p, 0, 1, 1, 1, 1, 1, 2, p, p, None), "format")
    bad(lib.csn_q8_pack(p, 0, -1, 1, 1, 1, 1, 0, p, p, None), "sizes")
    bad(lib.csn_q8_pack(p, 0, 1 << 40, 1 << 40, 1 << 40, 1, 1, 0, p, p, None), "sizes")
    bad(lib.csn_q8_pack(p, 0, 1, 4, 4, 0, -4, 0, p, p, None), "strides")
    bad(lib.csn_q8_pack(None, 0, 1, 4, 4, 0, 4, 0, p, p, None), "null")
    bad(lib.csn_q8_pack(C.c_void_p(4098), 0, 1, 4, 4, 0, 4, 0, p, p, None), "misaligned")
    bad(lib.csn_q8_unpack(p, p, 0, 4, 4, None, 0, None), "null")
    bad(lib.csn_q8_unpack(p, p, 0, -4, 4, p, 0, None), "sizes")

    def desc(**k):
        d = N.NormDesc()
        d.layout, d.dtype, d.outer, d.channels, d.inner, d.eps, d.format = 1, 0, 4, 8, 1, 1e-5, 0
        for a, v in k.items():
            setattr(d, a, v)
        return C.byref(d)
    fwd = lambda d, **k: lib.csn_layer_norm_forward(d, k.get("x", p), k.get("so", 8), 0, None, None, k.get("y", p), None, None,
                                                    k.get("codes"), k.get("exps"), None)
    bad(fwd(None), "null")
    bad(fwd(desc(layout=2)), "layout")
    bad(fwd(desc(dtype=2)), "dtype")
    bad(fwd(desc(channels=0)), "channels")
    bad(fwd(desc(channels=(1 << 24) + 1)), "channels")
    bad(fwd(desc(outer=-1)), "sizes")
    bad(fwd(desc(inner=2)), "inner")
    bad(fwd(desc(eps=0.0)), "eps")
    bad(fwd(desc(eps=float("inf"))), "eps")
    bad(fwd(desc(outer=1 << 45)), "elements")
    bad(fwd(desc(), so=-8), "strides")
    bad(fwd(desc(), x=None), "null")
    bad(fwd(desc(), y=C.c_void_p(4097)), "misaligned")
    bad(fwd(desc(), codes=p), "exponents")
    bad(fwd(desc(format=9), codes=p, exps=p), "format")
    assert lib.csn_layer_norm_workspace_bytes(desc(eps=0.0)) == 0

    def bwd(d, **k):
        return lib.csn_layer_norm_backward(d, k.get("dy", p), 8, 0, k.get("x", p), 8, 0, k.get("codes"), k.get("exps"), k.get("mean", p), p,
                                           None, k.get("dx", p), k.get("dw", p), p, k.get("ws", p), k.get("nws", 1 << 40), None)
    bad(bwd(desc(), dy=None), "null")
    bad(bwd(desc(), mean=None), "null")
    bad(bwd(desc(), x=None), "null")
    bad(bwd(desc(), codes=p, exps=p), "not both")
    bad(bwd(desc(), dx=C.c_void_p(4098)), "misaligned")
    need = lib.csn_layer_norm_workspace_bytes(desc())
    if need:
        bad(bwd(desc(), nws=need - 1), "workspace")
        bad(bwd(desc(), ws=None), "workspace")

    def pdesc(**k):
        d = N.ProductDesc()
        d.layout, d.dtype, d.format, d.outer, d.inner, d.cin, d.cout = 1, 0, 0, 4, 1, 8, 8
        for a, v in k.items():
            setattr(d, a, v)
        return C.byref(d)
    prod = lambda d, **k: lib.csn_product_weight_grad(d, k.get("dy", p), 8, 0, p, p, k.get("dw", p), None, k.get("ws", p), k.get("nws", 1 << 40), None)
    bad(prod(None), "null")
    bad(prod(pdesc(cin=0)), "channels")
    bad(prod(pdesc(format=3)), "format")
    bad(prod(pdesc(inner=3)), "inner")
    bad(prod(pdesc(), dy=None), "null")
    bad(prod(pdesc(), dw=None), "null")
    need = lib.csn_product_weight_grad_workspace_bytes(pdesc())
    if need:
        bad(prod(pdesc(), nws=need - 1), "workspace")


# ---- 8-bit checkpoints of whole forwards (CSNet.set_train_checkpoints) -------------------------------------------------------
def _net(lib, device, manifest, act_dtype, B):
    import parity_cases as P
    m, _ = P.make_model(lib, manifest, device)
    m.set_train_act_dtype(act_dtype)
    m.train()
    m.set_batchsize(B)
    m.clear_flops()
    m.flops_hook(1.0)
    return m


def check_plan_checkpoint(lib, device, manifest, act_dtype, fmt, B=2, size=32):
    """save + restore puts the packed values of every stored activation and raw convolution output where the tensors were, and the
    backward needs nothing else: with the whole workspace overwritten in between it gives the same bits."""
    from oracle import inputs as I
    m = _net(lib, device, manifest, act_dtype, B)
    f = {"int8": N.Q8_INT8, "e4m3": N.Q8_E4M3}[fmt]
    x = torch.from_numpy(I.randn_batch(31, B, size, size)).to(device)
    eng = m.engine_for(x, train=True)
    eng.workspace.fill_(255)                                   # NaN in every type: what the forward does not write is told apart
    y, _ = m._train_forward_raw(x)
    dy = gradient(tuple(y.shape), torch.float32, 1, device)
    acts = [i for i in range(1, eng.n_acts)]
    before = {}
    for i in acts:
        for what in ("act", "z"):
            try:
                before[i, what] = eng.train_probe(i, what)
            except ValueError:
                pass
    buf = eng.checkpoint_save(f)
    small = sum(t.numel() for t in before.values())
    assert buf.numel() < 2.2 * small + (1 << 24)              # one byte an element (pooled copies included) + the packed tables
    eng.checkpoint_restore(buf, f)
    changed = 0
    for (i, what), t in before.items():
        q = T.q8_pack(m._lib or N.load(), t, fmt, start_dim=2)
        v, now = T.q8_unpack(m._lib or N.load(), q), eng.train_probe(i, what)
        if bool(torch.isnan(t).all()):
            assert what == "act"                              # (an activation that its consumer forms on load is not stored)
            continue
        changed += 1
        assert same(now.cpu(), v.cpu())
    assert changed > 0.6 * len(before)
    g1 = m._train_backward_raw(x, dy, 0.7).clone()
    eng.workspace.fill_(255)                                   # NaN in every type
    eng.checkpoint_restore(buf, f)
    g2 = m._train_backward_raw(x, dy, 0.7)
    assert bool(torch.isfinite(g2).all()) and torch.equal(g1, g2)
    return g1


def check_two_forwards_one_backward(lib, device, manifest, act_dtype, fmt, B=2, size=32, quick=False):
    """A loss over two forwards: the newer one's gradients are exact, the older one's those of its checkpoint, whichever goes first;
    a lone forward is not touched.  quick: the two backwards in autograd's order alone."""
    from oracle import inputs as I
    xs = [torch.from_numpy(I.randn_batch(s, B, size, size)).to(device) for s in (31, 32)]
    f = {"int8": N.Q8_INT8, "e4m3": N.Q8_E4M3}[fmt]

    def lone(x, through_checkpoint):
        m = _net(lib, device, manifest, act_dtype, B)
        y, _ = m._train_forward_raw(x)
        if through_checkpoint:
            eng = m.engine_for(x, train=True)
            eng.checkpoint_restore(eng.checkpoint_save(f), f)
        return m._train_backward_raw(x, gradient(tuple(y.shape), torch.float32, 1, device), 0.0).clone()
    ck0, exact1 = lone(xs[0], True), lone(xs[1], False)

    def flat(m):
        out = torch.zeros_like(ck0)
        for n, p in m.named_parameters():
            o = m._arena.offsets[n]
            out[o:o + p.numel()] = p.grad.reshape(-1)
        return out

    def fresh():
        m = _net(lib, device, manifest, act_dtype, B)
        m.set_train_checkpoints(fmt)
        return m
    dy = gradient((B, 1, size, size), torch.float32, 1, device)
    if quick:
        m = fresh()
        a, b = (m(x) for x in xs)
        b.backward(dy)
        assert torch.equal(flat(m), exact1)
        m.zero_grad(set_to_none=True)
        a.backward(dy)
        assert torch.equal(flat(m), ck0)
        return
    exact0, ck1 = lone(xs[0], False), lone(xs[1], True)
    m = fresh()                                                # one forward, one backward
    m(xs[0]).backward(dy)
    assert torch.equal(flat(m), exact0)
    for order in ((0, 1), (1, 0)):
        m = fresh()
        ys = [m(x) for x in xs]
        got = []
        for k in order:
            m.zero_grad(set_to_none=True)
            ys[k].backward(dy, retain_graph=True)
            got.append(flat(m))
        want = [ck0, exact1] if order == (0, 1) else [exact1, ck0]
        if order == (0, 1):                                    # the newer forward gave way to the older one's backward
            want = [ck0, ck1]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        m.zero_grad(set_to_none=True)
        ys[0].backward(dy)                                     # a checkpoint may be used again
        assert torch.equal(flat(m), ck0)
    m = fresh()                                                # one loss over both: autograd's own order, gradients added
    a, b = (m(x) for x in xs)
    torch.autograd.backward([a, b], [dy, dy])
    assert torch.equal(flat(m), exact1 + ck0) or torch.equal(flat(m), ck0 + ck1)
    m = fresh()                                                # a forward whose graph is dropped saves nothing
    a = m(xs[0])
    del a
    b = m(xs[1])
    assert m.engine_for(xs[1], train=True).waiting().checkpoint is None
    b.backward(dy)
    assert torch.equal(flat(m), exact1)


def check_waiting_forwards_refuse(lib, device, manifest, B=1, size=16):
    """Backwards whose forward's tensors or parameters are no longer there: refused, never wrong."""
    from oracle import inputs as I
    xs = [torch.from_numpy(I.randn_batch(s, B, size, size)).to(device) for s in (31, 32)]
    m = _net(lib, device, manifest, "fp32", B)
    m.set_train_checkpoints("int8")
    a = m(xs[0])
    m.set_train_checkpoints(None)
    b = m(xs[1])                                               # keeps no checkpoint; its tensors make room for a's
    a.sum().backward()
    with pytest.raises(RuntimeError, match="newer"):
        b.sum().backward()
    m.set_train_checkpoints("e4m3")
    c = m(xs[0])
    with torch.no_grad():
        next(m.parameters()).mul_(1.0)
    with pytest.raises(RuntimeError, match="in-place change"):
        c.sum().backward()
