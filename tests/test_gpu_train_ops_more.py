"""Further checks of the training operators beside the plan on the GPU."""
import pytest
import torch

import train_ops_cases as K
import train_ops_more as M
from sod100k_amd import _native as N, train_ops as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.fail("the GPU suite needs a ROCm device")
    return N.load()


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape,dim", M.CONSTANT)
def test_gpu_constant_tokens(lib, shape, dim, dtype):
    M.check_constant_tokens(lib, DEV, shape, dim, dtype)


@pytest.mark.parametrize("shape,dim", [((3, 100), -1), ((2, 40, 3, 5), 1)])
def test_gpu_nan_statistics(lib, shape, dim):
    M.check_nan_statistics(lib, DEV, shape, dim)


def test_gpu_without_gradients(lib, monkeypatch):
    M.check_without_gradients(lib, DEV, monkeypatch)


def test_gpu_captured_without_gradients(lib):
    """An inference pass of the differentiable forms, parameters included, captured and replayed between eager work."""
    x = K.activations((40, 64), torch.bfloat16, 1, DEV)
    w, b = (torch.nn.Parameter(p) for p in K.params(64, 1, DEV))
    W = torch.nn.Parameter(torch.randn(32, 64, generator=torch.Generator().manual_seed(2)).to(DEV))

    def run():
        with torch.no_grad():
            return T.product(T.layer_norm(x, w, b, checkpoint="int8"), W)
    want = run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(run(), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_gpu_frozen_norm(lib, monkeypatch):
    M.check_frozen_norm(lib, DEV, monkeypatch)


def test_gpu_autocast(lib):
    M.check_autocast(lib, DEV)


def test_gpu_refusals_of_workspaces(lib):
    M.check_refusals_of_workspaces(lib)


def test_gpu_outputs_end_where_they_end(lib):
    M.check_outputs_end_where_they_end(lib, DEV)


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape", M.MANY_ROWS)
def test_gpu_many_rows(lib, shape, dtype):
    M.check_many_tokens(lib, DEV, shape, -1, dtype)


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape", M.MANY_MAPS)
def test_gpu_many_maps(lib, shape, dtype):
    M.check_many_tokens(lib, DEV, shape, 1, dtype)


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("gap", [-128, 64])
def test_gpu_far_channels(lib, dtype, gap):
    """Channels 2^26 elements apart: a lane's 32-bit byte offsets just hold them (gap -128), or the simple kernels take over."""
    far = (1 << 26) + gap
    base = torch.empty((8, far), dtype=dtype, device=DEV)
    x = base.view(1, 8, far)[:, :, 100:170]
    x.copy_(K.activations((1, 8, 70), dtype, 1, DEV, rows=False))
    assert x.stride(1) == far and T._view(x, False)[0].data_ptr() == x.data_ptr()
    w, b = K.params(8, 1, DEV)
    dy = K.gradient((1, 8, 70), dtype, 1, DEV)
    _, mean, rstd, _ = K.check_norm_forward(lib, x, w, b, 1)
    K.check_norm_backward(lib, dy, x, mean, rstd, w, 1)
    for fmt in K.FORMATS:
        q = K.check_norm_forward(lib, x, w, b, 1, checkpoint=fmt)[3]
        K.check_pack(lib, x, fmt, 2)
        K.check_norm_backward(lib, dy, x, mean, rstd, w, 1, q=q)
    x.copy_(dy)                                    # the gradient lies far apart
    x2 = K.activations((1, 8, 70), dtype, 2, DEV, rows=False)
    _, mean, rstd, q = T.layer_norm_forward(lib, x2, w, b, dim=1, checkpoint="int8")
    K.check_norm_backward(lib, x, x2, mean, rstd, w, 1)
    dw, db = T.product_weight_grad(lib, x, q, dim=1)
    ref = T.product_weight_grad(lib, dy, q, dim=1)
    assert torch.equal(dw, ref[0]) and torch.equal(db, ref[1])


def test_gpu_maps_beyond_32_bits(lib):
    """Maps of more than 2^31 elements: the last image's results are those of that image alone."""
    shape = (280, 256, 176, 176)
    x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    last = K.activations((1,) + shape[1:], torch.bfloat16, 1, DEV, rows=False)
    dlast = K.gradient((1,) + shape[1:], torch.bfloat16, 1, DEV)
    x[-1:] = last
    w, b = K.params(256, 1, DEV)
    y, mean, rstd, q = T.layer_norm_forward(lib, x, w, b, dim=1, checkpoint="int8")
    one = T.layer_norm_forward(lib, last, w, b, dim=1, checkpoint="int8")
    assert torch.equal(y[-1:], one[0]) and torch.equal(mean[-1:], one[1]) and torch.equal(rstd[-1:], one[2])
    assert torch.equal(q.codes[-1:], one[3].codes) and torch.equal(q.scales[-1:], one[3].scales) and not bool(q.codes[:-1].any())
    y.zero_()
    y[-1:] = dlast
    for src, alone in ((x, last), (q, one[3])):
        dx, dw, db = T.layer_norm_backward(lib, y, src, mean, rstd, w, dim=1)
        ref = T.layer_norm_backward(lib, dlast, alone, one[1], one[2], w, dim=1)
        assert torch.equal(dx[-1:], ref[0])
        for s, t, a in zip((dw, db), ref[1:], ((dlast.float() * (last.float() - one[1][:, None]) * one[2][:, None]).abs(), dlast.float().abs())):
            assert bool(((s - t).abs() <= 2 * 1024 * K.U * a.sum((0, 2, 3))).all())
        del dx
    dW, dB = T.product_weight_grad(lib, y[:, :9], q, dim=1)
    ref, rb = T.product_weight_grad(lib, dlast[:, :9], one[3], dim=1)
    v = T.q8_unpack(lib, one[3]).flatten(2)[0].abs()
    bound = 2 * 1024 * K.U * (dlast[0, :9].float().abs().flatten(1) @ v.t())
    assert bool(((dW - ref).abs() <= bound).all()) and torch.allclose(dB, rb, rtol=0, atol=2 * 1024 * K.U * float(dlast[0, :9].abs().float().flatten(1).sum(1).max()))


def test_gpu_planes_beyond_29_bits(lib):
    """Planes of more than 2^29 pixels (the simple kernels): the last pixels' results are those of the tail alone."""
    n, c = (1 << 29) + 33, 2
    x = torch.zeros((1, c, n), dtype=torch.bfloat16, device=DEV)
    tail = K.activations((1, c, 64), torch.bfloat16, 1, DEV, rows=False)
    x[:, :, -64:] = tail
    y, mean, rstd, _ = T.layer_norm_forward(lib, x, dim=1)
    K.check_norm_forward(lib, tail, None, None, 1)
    t = tail[0].double()
    m = t.mean(0)
    r = 1 / torch.sqrt(((t - m) ** 2).mean(0) + 1e-5)
    assert bool(((mean[0, -64:].double() - m).abs() <= 64 * K.U * t.abs().amax(0)).all())
    want = (t - m) * r
    assert bool(((y[0, :, -64:].double() - want).abs() <= (64 * K.U + 64 * K.U * t.abs().amax(0) * r) + K.HALF[torch.bfloat16] * want.abs()).all())
    assert not bool(y[:, :, :-64].any()) and not bool(mean[0, :-64].any())
