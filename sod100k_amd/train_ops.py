"""Training operators beside the plan: layer norm, 8-bit checkpoints of activations, product gradients.

Free operators of ``include/csnet_hip.h`` on torch tensors.  Like the functions of ``engine.py`` each takes the bound library
first; PyTorch supplies device memory and the current stream, all arithmetic of the kernels happens in libcsnet_hip.so.  float32
and bfloat16 tensors; weights, statistics and their gradients are float32.  A ``dim`` argument names the channel axis: ``1`` for
planar maps ``[B, C, ...]`` (the framework's layout), ``-1`` for rows of tokens ``[..., C]``.

``layer_norm`` and ``product`` at the end of the file are the differentiable forms.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _native as N

_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16}
_FORMATS = {"int8": N.Q8_INT8, "e4m3": N.Q8_E4M3}


class Q8(NamedTuple):
    """8-bit checkpoint of a tensor: ``codes`` (uint8, the tensor's shape) and ``scales``, one power-of-two exponent byte per 32
    elements of the axes from ``start_dim`` on, which count as one (``2`` for planar maps, ``-1`` for rows)."""
    codes: torch.Tensor
    scales: torch.Tensor
    format: str
    start_dim: int


def _format(fmt: str) -> int:
    if fmt not in _FORMATS:
        raise ValueError(f"unknown checkpoint format {fmt!r} (one of {sorted(_FORMATS)})")
    return _FORMATS[fmt]


def _dtype(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what}: float32 or bfloat16 expected, got {t.dtype}")
    return _DTYPES[t.dtype]


def _same_device(lib: C.CDLL, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """The tensors' one device.  The product library works on ROCm tensors only (no CPU fallback)."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    if (dev.type == "cuda") != (lib is N._lib):
        raise RuntimeError(f"this library does not work on {dev.type} tensors (the HIP path is ROCm only: there is no CPU fallback)")
    return dev


def _launch(lib: C.CDLL, dev: torch.device, what: str, *args) -> None:
    """Call entry point ``what`` with ``args`` and the current stream of ``dev``, which is made current if another device is (a
    launch goes to the device that is current)."""
    fn = getattr(lib, what)
    if dev.type != "cuda":
        st = fn(*args, None)
    elif torch.cuda.current_device() == dev.index:
        st = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if st:
        N.check(lib, st, what)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _channel_axis(dim: int, ndim: int) -> bool:
    """True for rows (the channels are the last axis), False for planar maps (axis 1 of at least three)."""
    if not -ndim <= dim < ndim:
        raise ValueError(f"dim {dim} out of range for {ndim} axes")
    if dim % ndim == ndim - 1:
        return True
    if dim % ndim == 1:
        return False
    raise ValueError("the channel axis is the last one (rows) or axis 1 (planar maps)")


def _view(x: torch.Tensor, rows: bool) -> Tuple[torch.Tensor, int, int]:
    """(tensor, outer stride, channel stride) of x as [tokens][C] or [B][C][pixels] with consecutive innermost elements; slices of
    wider tensors are taken as they lie, anything else is copied."""
    if x.is_contiguous():
        ch = x.shape[-1] if rows else x.shape[1]
        return (x, ch, 0) if rows else (x, x.numel() // x.shape[0], x.numel() // (x.shape[0] * ch))
    shape, stride = x.shape, x.stride()
    end, n = (len(shape) - 1, -1) if rows else (len(shape), 1)     # the axes [0, end) / [2, end) have to lie as one, n apart (-1: any)
    if rows and shape[-1] > 1 and stride[-1] != 1:
        return x.contiguous(), shape[-1], 0
    so = 0
    for d in range(end - 1, -1 if rows else 1, -1):
        if shape[d] > 1:
            if n == -1:
                n = so = stride[d]
            elif stride[d] != n:
                return _view(x.contiguous(), rows)
            n *= shape[d]
    if rows:
        return x, so, 0
    return x, stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0


def _blocks(cols: int) -> int:
    return -(-cols // N.Q8_BLOCK)


def _scales_shape(shape, start_dim: int) -> Tuple[int, ...]:
    if start_dim == -1:
        return tuple(shape[:-1]) + (_blocks(shape[-1]),)
    return tuple(shape[:start_dim]) + (_blocks(math.prod(shape[start_dim:])),)


def _check_q8(q: Q8) -> int:
    f = _format(q.format)
    if q.codes.dtype != torch.uint8 or q.scales.dtype != torch.uint8:
        raise TypeError("codes and scales of a checkpoint are uint8")
    if not q.codes.is_contiguous() or not q.scales.is_contiguous():
        raise ValueError("codes and scales of a checkpoint are contiguous")
    if q.start_dim not in (2, -1) or q.codes.dim() < (3 if q.start_dim == 2 else 1):
        raise ValueError("a checkpoint's blocks run along the last axis (start_dim -1) or over a map's pixels (start_dim 2)")
    if tuple(q.scales.shape) != _scales_shape(q.codes.shape, q.start_dim):
        raise ValueError(f"scales of shape {tuple(q.scales.shape)}, expected {_scales_shape(q.codes.shape, q.start_dim)}")
    return f


def _q8_rows(q: Q8) -> Tuple[int, int]:
    cols = math.prod(q.codes.shape[q.start_dim:])
    return (q.codes.numel() // cols if cols else 0), cols


def q8_pack(lib: C.CDLL, x: torch.Tensor, format: str = "int8", start_dim: int = -1) -> Q8:
    """8-bit checkpoint of ``x`` ("int8" or "e4m3").  The axes from ``start_dim`` on form the rows that are cut into blocks of 32:
    ``2`` for planar maps [B, C, ...], ``-1`` for rows [..., C]."""
    f, dt = _format(format), _dtype(x, "q8_pack")
    dev = _same_device(lib, x)
    if start_dim not in (2, -1) or x.dim() < (3 if start_dim == 2 else 1):
        raise ValueError("start_dim is -1 (the last axis) or 2 (the pixels of planar maps [B, C, ...])")
    rows = start_dim == -1
    codes = x.new_empty(x.shape, dtype=torch.uint8)
    scales = x.new_empty(_scales_shape(x.shape, start_dim), dtype=torch.uint8)
    if x.numel():
        v, so, sc = _view(x, rows)
        ch = x.shape[-1] if rows else x.shape[1]
        o, r, c, s0, s1 = (1, x.numel() // ch, ch, 0, so) if rows else (x.shape[0], ch, x.numel() // (x.shape[0] * ch), so, sc)
        _launch(lib, dev, "csn_q8_pack", v.data_ptr(), dt, o, r, c, s0, s1, f, codes.data_ptr(), scales.data_ptr())
    return Q8(codes, scales, format, start_dim)


def q8_unpack(lib: C.CDLL, q: Q8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of a checkpoint as a dense float32 or bfloat16 tensor (both hold them exactly)."""
    f = _check_q8(q)
    dev = _same_device(lib, q.codes, q.scales)
    y = q.codes.new_empty(q.codes.shape, dtype=dtype)
    dt = _dtype(y, "q8_unpack")
    if y.numel():
        rows, cols = _q8_rows(q)
        _launch(lib, dev, "csn_q8_unpack", q.codes.data_ptr(), q.scales.data_ptr(), f, rows, cols, y.data_ptr(), dt)
    return y


def _param(t: Optional[torch.Tensor], channels: int, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: float32 expected, got {t.dtype}")
    if tuple(t.shape) != (channels,):
        raise ValueError(f"{what}: shape ({channels},) expected, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _norm_desc(rows: bool, dt: int, shape, eps: float, fmt: int) -> N.NormDesc:
    if rows:
        return N.NormDesc(N.LAYOUT_ROWS, dt, math.prod(shape[:-1]), shape[-1], 1, eps, fmt)
    return N.NormDesc(N.LAYOUT_PLANAR, dt, shape[0], shape[1], math.prod(shape[2:]), eps, fmt)


def _dense_like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def layer_norm_forward(lib: C.CDLL, x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       dim: int = -1, eps: float = 1e-5, checkpoint: Optional[str] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, Optional[Q8]]:
    """``(y, mean, rstd, checkpoint)`` of the layer norm over axis ``dim``: ``y`` dense in x's dtype, the statistics float32 with
    x's shape without that axis, and, with ``checkpoint`` "int8" / "e4m3", the 8-bit checkpoint of x written in the same pass
    (else None)."""
    dt = _dtype(x, "layer_norm")
    rows = _channel_axis(dim, x.dim())
    ch = x.shape[-1] if rows else x.shape[1]
    weight, bias = _param(weight, ch, "weight"), _param(bias, ch, "bias")
    dev = _same_device(lib, x, weight, bias)
    fmt = _format(checkpoint) if checkpoint is not None else 0
    d = _norm_desc(rows, dt, x.shape, eps, fmt)
    y = _dense_like(x)
    sshape = x.shape[:-1] if rows else x.shape[:1] + x.shape[2:]
    mean, rstd = x.new_empty((2,) + sshape, dtype=torch.float32).unbind()   # (one allocation: the host's share of a small call)
    q = codes = scales = None
    if checkpoint is not None:
        start = -1 if rows else 2
        q = Q8(x.new_empty(x.shape, dtype=torch.uint8), x.new_empty(_scales_shape(x.shape, start), dtype=torch.uint8), checkpoint, start)
        if x.numel():
            codes, scales = q.codes.data_ptr(), q.scales.data_ptr()
    v, so, sc = _view(x, rows) if x.numel() else (x, 0, 0)
    _launch(lib, dev, "csn_layer_norm_forward", C.byref(d), v.data_ptr(), so, sc, _ptr(weight), _ptr(bias), y.data_ptr(),
            mean.data_ptr(), rstd.data_ptr(), codes, scales)
    return y, mean, rstd, q


def layer_norm_backward(lib: C.CDLL, dy: torch.Tensor, x: Union[torch.Tensor, Q8], mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, dim: int = -1, param_grads: bool = True
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dx, dweight, dbias)`` of a layer norm from its input ``x`` -- the tensor or its checkpoint -- and the statistics of the
    forward.  ``dx`` is dense in dy's dtype, the parameter gradients float32; ``param_grads=False`` leaves them out (None): a frozen
    norm's backward is one launch."""
    dt = _dtype(dy, "layer_norm")
    rows = _channel_axis(dim, dy.dim())
    ch = dy.shape[-1] if rows else dy.shape[1]
    weight = _param(weight, ch, "weight")
    q = x if isinstance(x, Q8) else None
    fmt = _check_q8(q) if q is not None else 0
    src = q.codes if q is not None else x
    if src.shape != dy.shape:
        raise ValueError(f"dy of shape {tuple(dy.shape)}, the input has {tuple(src.shape)}")
    if q is None and x.dtype != dy.dtype:
        raise TypeError(f"dy is {dy.dtype}, the input {x.dtype}")
    if q is not None and q.start_dim != (-1 if rows else 2):
        raise ValueError("the checkpoint was packed for the other layout")
    sshape = tuple(dy.shape[:-1] if rows else dy.shape[:1] + dy.shape[2:])
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or tuple(t.shape) != sshape:
            raise ValueError(f"{what}: float32 of shape {sshape} expected, got {t.dtype} {tuple(t.shape)}")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dev = _same_device(lib, dy, src, q.scales if q is not None else None, mean, rstd, weight)
    d = _norm_desc(rows, dt, dy.shape, 1.0, fmt)
    dx = _dense_like(dy)
    dweight = dbias = ws = None
    nbytes = 0
    if param_grads:
        dweight = dy.new_empty((ch,), dtype=torch.float32)
        dbias = dy.new_empty((ch,), dtype=torch.float32)
        nbytes = lib.csn_layer_norm_workspace_bytes(C.byref(d))
        ws = dy.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    vd, dso, dsc = _view(dy, rows) if dy.numel() else (dy, 0, 0)
    vx, so, sc, codes, scales = None, 0, 0, None, None
    if dy.numel():
        if q is None:
            vx, so, sc = _view(x, rows)
        else:
            codes, scales = q.codes.data_ptr(), q.scales.data_ptr()
    _launch(lib, dev, "csn_layer_norm_backward", C.byref(d), vd.data_ptr(), dso, dsc, _ptr(vx), so, sc, codes, scales, mean.data_ptr(),
            rstd.data_ptr(), _ptr(weight), dx.data_ptr(), _ptr(dweight), _ptr(dbias), _ptr(ws), nbytes)
    return dx, dweight, dbias


def product_weight_grad(lib: C.CDLL, dy: torch.Tensor, q: Q8, dim: int = -1) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(dweight [Cout, Cin], dbias [Cout])``, float32, of a 1x1 convolution (``dim=1``) or linear layer (``dim=-1``) from the
    gradient of its output and the checkpoint of its input."""
    dt = _dtype(dy, "product_weight_grad")
    fmt = _check_q8(q)
    rows = _channel_axis(dim, dy.dim())
    if q.start_dim != (-1 if rows else 2):
        raise ValueError("the checkpoint was packed for the other layout")
    xs, ds = tuple(q.codes.shape), tuple(dy.shape)
    if (xs[:-1] != ds[:-1]) if rows else (len(xs) != len(ds) or xs[:1] + xs[2:] != ds[:1] + ds[2:]):
        raise ValueError(f"dy of shape {ds} does not belong to an input of shape {xs}")
    dev = _same_device(lib, dy, q.codes, q.scales)
    nd = _norm_desc(rows, dt, ds, 1.0, fmt)
    d = N.ProductDesc()
    d.layout, d.dtype, d.format, d.outer, d.inner = nd.layout, dt, fmt, nd.outer, nd.inner
    d.cin, d.cout = (xs[-1], ds[-1]) if rows else (xs[1], ds[1])
    dweight = dy.new_empty((d.cout, d.cin), dtype=torch.float32)
    dbias = dy.new_empty((d.cout,), dtype=torch.float32)
    nbytes = lib.csn_product_weight_grad_workspace_bytes(C.byref(d))
    ws = dy.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    v, so, sc = _view(dy, rows) if dy.numel() else (dy, 0, 0)
    _launch(lib, dev, "csn_product_weight_grad", C.byref(d), v.data_ptr(), so, sc, q.codes.data_ptr(), q.scales.data_ptr(),
            dweight.data_ptr(), dbias.data_ptr(), _ptr(ws), nbytes)
    return dweight, dbias


# ---- differentiable forms -------------------------------------------------------------------------------------------------
def _refuse_capture() -> None:
    """Autograd inside a stream capture depends on what other graphs of the same leaves live on (their accumulation nodes keep the
    stream they were made on, and the engine's wait for it breaks the capture): the raw forms above are for captures."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("layer_norm / product with gradients inside a stream capture: capture the *_forward / *_backward / "
                           "*_weight_grad functions instead")


def _records(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd records an operator on these tensors: where it does not, nothing is kept for a backward pass."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lib, x, weight, bias, dim, eps, checkpoint):
        _refuse_capture()
        y, mean, rstd, q = layer_norm_forward(lib, x, weight, bias, dim=dim, eps=eps, checkpoint=checkpoint)
        ctx.lib, ctx.dim = lib, dim
        if q is None:
            ctx.save_for_backward(mean, rstd, weight, x)
            ctx.q = None
        else:
            ctx.save_for_backward(mean, rstd, weight, q.codes, q.scales)
            ctx.q = (q.format, q.start_dim)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture()
        mean, rstd, weight, *src = ctx.saved_tensors
        x = src[0] if ctx.q is None else Q8(src[0], src[1], *ctx.q)
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(ctx.lib, dy, x, mean, rstd, weight, dim=ctx.dim, param_grads=need[2] or need[3])
        return None, dx if need[1] else None, dw if need[2] else None, db if need[3] else None, None, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, dim: int = -1,
               eps: float = 1e-5, checkpoint: Optional[str] = None, lib: Optional[C.CDLL] = None) -> torch.Tensor:
    """Differentiable layer norm over axis ``dim``.  ``checkpoint`` ("int8" / "e4m3") keeps x for the backward in 8 bits instead of
    the tensor itself: the gradients are then those of the checkpoint's values.  Without gradients (``torch.no_grad()``) nothing is
    kept, and the call may be captured."""
    lib = lib or N.load()
    if not _records(x, weight, bias):
        if checkpoint is not None:
            _format(checkpoint)
        return layer_norm_forward(lib, x, weight, bias, dim=dim, eps=eps)[0]
    return _LayerNormFn.apply(lib, x, weight, bias, dim, eps, checkpoint)


def _product(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], rows: bool) -> torch.Tensor:
    """The forward product itself: one library matrix product in x's dtype, whatever autocast would make of it."""
    if torch.is_autocast_enabled(x.device.type):
        with torch.autocast(x.device.type, enabled=False):
            return _product(x, weight, bias, rows)
    w = weight.to(x.dtype)
    b = None if bias is None else bias.to(x.dtype)
    if rows:
        return torch.nn.functional.linear(x, w, b)
    y = torch.matmul(w, x.flatten(2).contiguous())
    if b is not None:
        y += b.view(1, -1, 1)
    return y.view(x.shape[:1] + (w.shape[0],) + x.shape[2:])


class _ProductFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lib, x, weight, bias, dim, checkpoint):
        _refuse_capture()
        rows = _channel_axis(dim, x.dim())
        y = _product(x, weight, bias, rows)
        ctx.lib, ctx.dim, ctx.rows = lib, dim, rows
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            q = q8_pack(lib, x, checkpoint, start_dim=-1 if rows else 2)
            ctx.q = (q.format, q.start_dim)
            ctx.save_for_backward(weight, q.codes, q.scales)
        else:
            ctx.save_for_backward(weight)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture()
        weight, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[1]:
            dx = _product(dy, weight.t().contiguous(), None, ctx.rows)
        if need[2] or need[3]:
            dw, db = product_weight_grad(ctx.lib, dy, Q8(*kept, *ctx.q), dim=ctx.dim)
        return None, dx, dw if need[2] else None, db if need[3] else None, None, None


def product(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, dim: int = -1, checkpoint: str = "int8",
            lib: Optional[C.CDLL] = None) -> torch.Tensor:
    """Differentiable 1x1 convolution over planar maps (``dim=1``) or linear layer over rows (``dim=-1``), weight [Cout, Cin], that
    keeps its input for the weight gradient as an 8-bit checkpoint.  The forward and the input gradient are exact library products
    in x's dtype; only the weight gradient sees the checkpoint's values.  Without gradients (``torch.no_grad()``) nothing is kept, and
    the call may be captured."""
    lib = lib or N.load()
    ch = x.shape[-1] if _channel_axis(dim, x.dim()) else x.shape[1]
    if weight.dim() != 2 or weight.shape[1] != ch or weight.dtype != torch.float32:
        raise ValueError(f"weight: float32 of shape (Cout, {ch}) expected, got {weight.dtype} {tuple(weight.shape)}")
    bias = _param(bias, weight.shape[0], "bias")
    _dtype(x, "product")
    _format(checkpoint)
    _same_device(lib, x, weight, bias)
    if not _records(x, weight, bias):
        return _product(x, weight, bias, _channel_axis(dim, x.dim()))
    return _ProductFn.apply(lib, x, weight, bias, dim, checkpoint)
