"""Cases that measure the training operators next to the plan: layer norm, 8-bit checkpoints, product gradients.

Four kinds of case, each one pass of what a training or serving program does with them:

``norm``        layer norm over the channels of planar maps (``layout="planar"``, B x C x H x W) or of token rows
                (``layout="rows"``, T x C): the forward alone, or the forward and the backward of a training step
``norm_q8``     the same training step with the input kept for the backward pass as an 8-bit checkpoint
``checkpoint``  an activation packed into 8 bits and unpacked again
``product``     weight and bias gradient of a 1x1 convolution or linear layer whose input is kept in 8 bits
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32
FMT_MAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZEOF = {"fp32": 4, "bf16": 2}


def listed():
    return [
        # one token through the norm in front of a head: all launch latency.  2048 = the widest feature level of the CSF network
        dict(name="norm_token", kind="norm", layout="rows", B=1, C=2048, H=1, W=1, dtype="bf16", train=False, slack=0),
        # a training step's norm over the tokens of 32 maps of 28 x 28, all parameters and activations in 32 bits
        dict(name="norm_rows", kind="norm", layout="rows", B=32, C=512, H=28, W=28, dtype="fp32", train=True, slack=0),
        # ... over the channels of the CSF network's finest feature level (batch 32 of 352 x 352 pictures)
        dict(name="norm_planar", kind="norm", layout="planar", B=32, C=256, H=88, W=88, dtype="bf16", train=True, slack=0),
        # three pictures of an odd size, 79 channels (the width of the fused head) cut out of a wider tensor
        dict(name="norm_ragged", kind="norm", layout="planar", B=3, C=79, H=37, W=53, dtype="fp32", train=True, slack=5),
        # a single picture's stage-1 map kept between its forward and backward
        dict(name="checkpoint_small", kind="checkpoint", layout="planar", B=1, C=40, H=56, W=56, dtype="fp32", fmt="int8"),
        # the finest maps of a training batch in the bf16 storage mode
        dict(name="checkpoint_large", kind="checkpoint", layout="planar", B=64, C=40, H=224, W=224, dtype="bf16", fmt="int8"),
        # maps whose planes end inside a block of 32
        dict(name="checkpoint_ragged", kind="checkpoint", layout="planar", B=17, C=60, H=27, W=31, dtype="bf16", fmt="e4m3"),
        # a token model's norm with 8-bit activations
        dict(name="norm_q8_rows", kind="norm_q8", layout="rows", B=16, C=1024, H=32, W=32, dtype="bf16", fmt="int8", slack=0),
        # the CSF network's second feature level, 32-bit activations, floating-point codes
        dict(name="norm_q8_planar", kind="norm_q8", layout="planar", B=16, C=512, H=44, W=44, dtype="fp32", fmt="e4m3", slack=0),
        # the CSF head's first 1x1 product, 256 -> 128 channels on 88 x 88 maps
        dict(name="product_planar", kind="product", layout="planar", B=32, C=256, O=128, H=88, W=88, dtype="bf16", fmt="int8"),
        # the widening product of a token model
        dict(name="product_rows", kind="product", layout="rows", B=16, C=1024, O=4096, H=32, W=32, dtype="bf16", fmt="int8"),
        # odd widths on small maps, gradients in 32 bits
        dict(name="product_ragged", kind="product", layout="planar", B=5, C=37, O=21, H=13, W=17, dtype="fp32", fmt="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_q8", "checkpoint", "product"])
    case = dict(kind=kind, layout=rng.choice(["planar", "rows"]), dtype=rng.choice(["fp32", "bf16"]))
    H = _log_int(rng, 1, 96)
    W = min(224, max(1, int(H * rng.uniform(0.6, 1.6))))
    B = _log_int(rng, 1, 32)
    C = _log_int(rng, 8 if kind.startswith("norm") else 1, 2048)      # (two or three channels normalise to +-1: all rounding)
    if rng.random() < 0.4:        # the widths of real models are multiples of 8 more often than not
        C = (C + 7) // 8 * 8
    while B * C * H * W > 60_000_000:
        if B > 1:
            B //= 2
        else:
            C = C // 2 + 1
    case.update(B=B, C=C, H=H, W=W)
    if kind == "norm":
        case.update(train=rng.random() < 0.7)
    else:
        case.update(fmt=rng.choice(["int8", "e4m3"]))
    if kind.startswith("norm"):
        case.update(slack=rng.choice([0, 0, 1, 8]))
    if kind == "product":
        O = _log_int(rng, 1, 4096)
        while B * O * H * W > 60_000_000 or B * O * H * W * C > 6e10:
            O = O // 2 + 1
            if O <= 2:
                break
        case.update(O=O)
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _shape(case, channels):
    if case["layout"] == "planar":
        return (case["B"], channels, case["H"], case["W"])
    return (case["B"] * case["H"] * case["W"], channels)


def _axis(case):
    return 1 if case["layout"] == "planar" else -1


def _start(case):
    return 2 if case["layout"] == "planar" else -1


def _per_channel(case, v):
    return v.view(1, -1, 1, 1) if case["layout"] == "planar" else v.view(1, -1)


def _activation(case, g, dev, channels):
    """Activations: every channel with its own offset and spread, a few channels far wider than the rest."""
    spread = torch.exp(0.5 * torch.randn(channels, generator=g, device=dev))
    spread = torch.where(torch.rand(channels, generator=g, device=dev) < 0.02, 8.0 * spread, spread)
    offset = 0.5 * torch.randn(channels, generator=g, device=dev)
    x = torch.randn(_shape(case, channels), generator=g, device=dev)
    x.mul_(_per_channel(case, spread)).add_(_per_channel(case, offset))
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["kind"] == "checkpoint":
        st["x"] = _activation(case, g, dev, case["C"])
        return st
    if case["kind"] == "product":
        x = _activation(case, g, dev, case["C"])
        dy = torch.randn(_shape(case, case["O"]), generator=g, device=dev).mul_(1e-2).to(dt)
        codes, scales = plain_pack(x, case["fmt"], _start(case))
        st.update(dy=dy, codes=codes, scales=scales)
        if own:
            from sod100k_amd import train_ops as T
            st["q"] = T.Q8(codes, scales, case["fmt"], _start(case))
        return st
    wide = _activation(case, g, dev, case["C"] + case["slack"])
    st["x"] = wide.narrow(_axis(case), case["slack"], case["C"]) if case["slack"] else wide
    st["weight"] = 1.0 + 0.2 * torch.randn(case["C"], generator=g, device=dev)
    st["bias"] = 0.2 * torch.randn(case["C"], generator=g, device=dev)
    if case.get("train", True):
        st["dy"] = torch.randn(_shape(case, case["C"]), generator=g, device=dev).mul_(1e-2).to(dt)
    return st


# ---- plain forms --------------------------------------------------------------------------------------------------------
def _blocks(x, start):
    """[..., columns] -> [..., blocks, 32] with zeros behind the last column."""
    flat = x.flatten(start) if start != -1 else x
    cols = flat.shape[-1]
    pad = -cols % BLOCK
    if pad:
        flat = torch.cat([flat, flat.new_zeros(flat.shape[:-1] + (pad,))], dim=-1)
    return flat.view(flat.shape[:-1] + (-1, BLOCK)), cols


def plain_pack(x, fmt, start):
    """Codes (one byte an element, in x's shape) and block exponents of x."""
    v, cols = _blocks(x.float(), start)
    finite = torch.isfinite(v)
    amax = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(-1)
    m, k = torch.frexp(amax)
    if fmt == "int8":            # 64 <= m 2^7 < 128; from 127.5 on it would round to 128
        e = torch.where(m * 128.0 >= 127.5, k - 6, k - 7)
    else:                        # 256 <= m 2^9 < 512; 464 still rounds (to even) to 448
        e = torch.where(m * 512.0 > 464.0, k - 8, k - 9)
    s = torch.where(amax > 0, e + 127, torch.full_like(e, 32)).clamp(min=32)
    t = torch.ldexp(v, (127 - s).unsqueeze(-1).to(torch.float32))
    t = torch.where(finite, t, torch.zeros_like(t))
    if fmt == "int8":
        c = torch.where(finite, torch.round(t), torch.full_like(t, -128.0)).to(torch.int8).view(torch.uint8)
    else:
        c = torch.where(finite, t, torch.full_like(t, float("nan"))).to(torch.float8_e4m3fn).view(torch.uint8)
    c = c.flatten(-2)[..., :cols].reshape(x.shape)
    return c.contiguous(), s.to(torch.uint8)


def plain_unpack(codes, scales, fmt, start):
    """The values that codes and exponents stand for, in 32 bits."""
    c, cols = _blocks(codes, start)
    if fmt == "int8":
        q = c.view(torch.int8).float()
        q = torch.where(q == -128.0, torch.full_like(q, float("nan")), q)
    else:
        q = c.view(torch.float8_e4m3fn).float()
    v = torch.ldexp(q, (scales.to(torch.int32) - 127).unsqueeze(-1).to(torch.float32))
    return v.flatten(-2)[..., :cols].reshape(codes.shape)


def _plain_norm(case, x, weight, bias):
    ax = _axis(case)
    mean = x.mean(ax, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(ax, keepdim=True) + EPS)
    y = d * rstd * _per_channel(case, weight) + _per_channel(case, bias)
    return y, mean, rstd


def _plain_norm_backward(case, dy, x, mean, rstd, weight):
    ax = _axis(case)
    dims = (0, 2, 3) if case["layout"] == "planar" else (0,)
    xh = (x - mean) * rstd
    g = dy * _per_channel(case, weight)
    c1 = g.mean(ax, keepdim=True)
    c2 = (g * xh).mean(ax, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    return dx, (dy * xh).sum(dims), dy.sum(dims)


def _plain(st):
    case = st["case"]
    if case["kind"] == "checkpoint":
        codes, scales = plain_pack(st["x"], case["fmt"], _start(case))
        return {"values": plain_unpack(codes, scales, case["fmt"], _start(case)).to(st["x"].dtype), "exponents": scales}
    if case["kind"] == "product":
        xv = plain_unpack(st["codes"], st["scales"], case["fmt"], _start(case))
        dy = st["dy"].float()
        if case["layout"] == "planar":
            dy = dy.flatten(2).transpose(0, 1).reshape(case["O"], -1)
            xv = xv.flatten(2).transpose(0, 1).reshape(case["C"], -1)
            return {"dweight": dy @ xv.t(), "dbias": dy.sum(1)}
        return {"dweight": dy.t() @ xv, "dbias": dy.sum(0)}
    x = st["x"].float()
    y, mean, rstd = _plain_norm(case, x, st["weight"], st["bias"])
    ax = _axis(case)
    out = {"y": y.to(st["x"].dtype), "mean": mean.squeeze(ax), "rstd": rstd.squeeze(ax)}
    if case.get("train", True):
        if case["kind"] == "norm_q8":
            codes, scales = plain_pack(st["x"], case["fmt"], _start(case))
            x = plain_unpack(codes, scales, case["fmt"], _start(case))
        dx, dw, db = _plain_norm_backward(case, st["dy"].float(), x, mean, rstd, st["weight"])
        out.update(dx=dx.to(st["x"].dtype), dweight=dw, dbias=db)
    return out


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _framework(st):
    from sod100k_amd import _native, train_ops as T
    lib = _native.load()
    case = st["case"]
    if case["kind"] == "checkpoint":
        q = T.q8_pack(lib, st["x"], case["fmt"], start_dim=_start(case))
        return {"values": T.q8_unpack(lib, q, st["x"].dtype), "exponents": q.scales}
    if case["kind"] == "product":
        dw, db = T.product_weight_grad(lib, st["dy"], st["q"], dim=_axis(case))
        return {"dweight": dw, "dbias": db}
    ckpt = case["fmt"] if case["kind"] == "norm_q8" else None
    y, mean, rstd, q = T.layer_norm_forward(lib, st["x"], st["weight"], st["bias"], dim=_axis(case), eps=EPS, checkpoint=ckpt)
    out = {"y": y, "mean": mean, "rstd": rstd}
    if case.get("train", True):
        dx, dw, db = T.layer_norm_backward(lib, st["dy"], st["x"] if ckpt is None else q, mean, rstd, st["weight"], dim=_axis(case))
        out.update(dx=dx, dweight=dw, dbias=db)
    return out


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    tokens = case["B"] * case["H"] * case["W"]
    n = tokens * case["C"]
    s = SIZEOF[case["dtype"]]
    if case["layout"] == "planar":
        nblk = case["B"] * case["C"] * (-(-case["H"] * case["W"] // BLOCK))
    else:
        nblk = tokens * (-(-case["C"] // BLOCK))
    if case["kind"] == "checkpoint":
        return {"bytes": 2 * (n * s + n + nblk), "flops": 3 * n}
    if case["kind"] == "product":
        m = tokens * case["O"]
        return {"bytes": m * s + n + nblk + 4 * case["O"] * (case["C"] + 1), "flops": 2 * m * case["C"] + m}
    if not case.get("train", True):
        return {"bytes": 2 * n * s + 8 * case["C"] + 8 * tokens, "flops": 8 * n}
    return {"bytes": 4 * n * s + 16 * case["C"] + 8 * tokens, "flops": 22 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_values(x, fmt, start):
    """Definition of the checkpoint: block by block the smallest power of two whose code of the largest value stays in range."""
    shape = x.shape
    rows = x.double().flatten(start) if start != -1 else x.double()
    cols = rows.shape[-1]
    n = -(-cols // BLOCK)
    full = torch.zeros(rows.shape[:-1] + (n * BLOCK,), dtype=torch.float64, device=x.device)
    full[..., :cols] = rows
    b = full.unflatten(-1, (n, BLOCK))

    def rounded(t):
        if fmt == "int8":
            return torch.round(t)
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3.0)
        return torch.round(t / step) * step

    amax = b.abs().amax(-1)
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -100))) - (7 if fmt == "int8" else 9)
    for _ in range(3):
        e = torch.where(rounded(amax * torch.exp2(-e)) > FMT_MAX[fmt], e + 1, e)
    e = e.clamp(min=-95.0)
    v = rounded(b * torch.exp2(-e).unsqueeze(-1)) * torch.exp2(e).unsqueeze(-1)
    return v.flatten(-2)[..., :cols].reshape(shape), e


def _tokens_last(case, t):
    """[channels, tokens] in 64 bits."""
    t = t.double()
    if case["layout"] == "planar":
        return t.movedim(1, 0).reshape(t.shape[1], -1)
    return t.t()


def _like(case, t, channels):
    if case["layout"] == "planar":
        return t.reshape(channels, case["B"], case["H"], case["W"]).movedim(0, 1)
    return t.t()


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "checkpoint":
        v, e = _exact_values(st["x"], case["fmt"], _start(case))
        return {"values": v, "exponents": (e + 127).to(torch.uint8)}
    if case["kind"] == "product":
        table = torch.arange(256, dtype=torch.int32, device=st["codes"].device)
        if case["fmt"] == "int8":
            table = torch.where(table < 128, table, table - 256).double()
        else:
            mant, ex = (table & 7).double(), ((table >> 3) & 15).double()
            table = torch.where(ex > 0, (8.0 + mant) * torch.exp2(ex - 10.0), mant * 2.0 ** -9) * (1.0 - 2.0 * (table >> 7).double())
        q = table[st["codes"].int()]
        q = q.flatten(2) if case["layout"] == "planar" else q
        each = torch.exp2(st["scales"].double() - 127.0).repeat_interleave(BLOCK, dim=-1)[..., :q.shape[-1]]
        x = _tokens_last(case, q * each)
        dy = _tokens_last(case, st["dy"])
        return {"dweight": dy @ x.t(), "dbias": dy.sum(1)}
    x = _tokens_last(case, st["x"])
    w, b = st["weight"].double()[:, None], st["bias"].double()[:, None]
    C = case["C"]
    mean = x.sum(0) / C
    var = ((x - mean) ** 2).sum(0) / C
    rstd = 1.0 / torch.sqrt(var + EPS)
    y = (x - mean) * rstd * w + b
    stat = (lambda t: t.reshape(case["B"], case["H"], case["W"])) if case["layout"] == "planar" else (lambda t: t)
    out = {"y": _like(case, y, C), "mean": stat(mean), "rstd": stat(rstd)}
    if case.get("train", True):
        if case["kind"] == "norm_q8":
            x = _tokens_last(case, _exact_values(st["x"], case["fmt"], _start(case))[0])
        dy = _tokens_last(case, st["dy"])
        xh = (x - mean) * rstd
        g = dy * w
        dx = rstd * (g - g.sum(0) / C - xh * ((g * xh).sum(0) / C))
        out.update(dx=_like(case, dx, C), dweight=(dy * xh).sum(1), dbias=dy.sum(1))
    return out
