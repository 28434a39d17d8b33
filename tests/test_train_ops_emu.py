"""Training operators beside the plan on the CPU emulation of their kernels (lane-exact mode: the device paths), and the refusals of
their Python and C entry points."""
import ctypes
import os

import pytest
import torch

import train_ops_cases as K
from sod100k_amd import _native as N, train_ops as T


@pytest.fixture(scope="module")
def lib(emu_lanes_lib):
    return emu_lanes_lib[0]


@pytest.mark.parametrize("fmt", K.FORMATS)
@pytest.mark.parametrize("dtype", K.DTYPES)
def test_emu_pack(lib, fmt, dtype):
    for i, (shape, start) in enumerate(K.PACK_SHAPES):
        K.check_pack(lib, K.activations(shape, dtype, i, rows=start == -1), fmt, start)
    K.check_pack(lib, K.block_edge_values(dtype), fmt, -1)


@pytest.mark.parametrize("fmt", K.FORMATS)
def test_emu_every_code(lib, fmt):
    q, want = K.every_code_once(fmt)
    for dtype in K.DTYPES:
        v = T.q8_unpack(lib, q, dtype)
        assert K.same(v.double(), want)


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape,dim", K.NORM_SHAPES)
def test_emu_norm(lib, shape, dim, dtype):
    rows = dim == -1
    x, dy = K.activations(shape, dtype, 1, rows=rows), K.gradient(shape, dtype, 1)
    w, b = K.params(shape[dim], 1)
    y, mean, rstd, _ = K.check_norm_forward(lib, x, w, b, dim)
    K.check_norm_forward(lib, x, None, None, dim)
    K.check_norm_backward(lib, dy, x, mean, rstd, w, dim)
    K.check_norm_backward(lib, dy, x, mean, rstd, None, dim)
    for fmt in K.FORMATS:
        y2, m2, r2, q = K.check_norm_forward(lib, x, w, b, dim, checkpoint=fmt)
        assert torch.equal(y, y2) and torch.equal(mean, m2) and torch.equal(rstd, r2)
        K.check_norm_backward(lib, dy, x, mean, rstd, w, dim, q=q)


@pytest.mark.parametrize("fmt", K.FORMATS)
@pytest.mark.parametrize("dtype", K.DTYPES)
def test_emu_product_gradient(lib, dtype, fmt):
    for i, (dims, cin, cout, dim) in enumerate(K.PRODUCT_SHAPES):
        x, dy = K.product_tensors(dims, cin, cout, dim, dtype, i)
        K.check_product(lib, dy, x, fmt, dim)


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_emu_slices_and_strides(lib, dtype):
    K.check_slices(lib, "cpu", dtype)


def test_emu_empty(lib):
    K.check_empty(lib, "cpu")


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_emu_bad_tokens_stay_alone(lib, dtype):
    K.check_bad_tokens_stay_alone(lib, "cpu", dtype)


def test_emu_constant_tokens_and_far_means(lib):
    K.check_constant_and_far(lib, "cpu")


def test_emu_determinism(lib):
    K.check_determinism(lib, "cpu")


def test_emu_gradients_against_differences(lib):
    K.check_against_differences(lib, "cpu")


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_emu_norm_and_product_together(lib, dtype):
    K.check_block_of_operators(lib, "cpu", dtype)


def test_refusals(lib):
    K.check_refusals(lib, "cpu")
    K.check_refusals_of_the_abi(lib)


def test_refusals_of_the_product_library():
    """The same refusals from the library that runs on the GPU: they are host code and follow no pointer."""
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("libcsnet_hip.so not built")
    K.check_refusals_of_the_abi(N.bind(ctypes.CDLL(N.LIB_PATH)))


def test_no_cpu_fallback(lib, monkeypatch):
    monkeypatch.setattr(N, "_lib", lib)      # the library that load() returned takes ROCm tensors only
    with pytest.raises(RuntimeError, match="ROCm"):
        T.layer_norm_forward(lib, torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="ROCm"):
        T.q8_pack(lib, torch.zeros(2, 4))


@pytest.mark.parametrize("act_dtype,fmt", [("fp32", "int8"), ("bf16", "e4m3")])
def test_emu_plan_checkpoint(lib, x2_manifest, act_dtype, fmt):
    K.check_plan_checkpoint(lib, torch.device("cpu"), x2_manifest, act_dtype, fmt)


def test_emu_two_forwards_one_backward(lib, x2_manifest):
    K.check_two_forwards_one_backward(lib, torch.device("cpu"), x2_manifest, "fp32", "int8", size=16, quick=True)


def test_emu_waiting_forwards_refuse(lib, x2_manifest):
    K.check_waiting_forwards_refuse(lib, torch.device("cpu"), x2_manifest)


def test_plan_checkpoint_refusals(lib, x2_manifest):
    import parity_cases as P
    m, _ = P.make_model(lib, x2_manifest, torch.device("cpu"))
    m.train()
    x = torch.zeros(1, 3, 32, 32)
    eng = m.engine_for(x, train=True)
    buf = torch.zeros(1 << 26, dtype=torch.uint8)
    p = buf.data_ptr() + (-buf.data_ptr() % 256)
    n = lib.csn_plan_checkpoint_bytes(eng.plan)
    ws = eng.workspace.data_ptr()
    for call in (lib.csn_plan_checkpoint_save, lib.csn_plan_checkpoint_restore):
        assert call(eng.plan, ws, 0, p, n, None) == 5                       # no forward yet
    m._train_forward_raw(x)
    for call in (lib.csn_plan_checkpoint_save, lib.csn_plan_checkpoint_restore):
        assert call(None, ws, 0, p, n, None) == 1 and call(eng.plan, None, 0, p, n, None) == 1
        assert call(eng.plan, ws, 2, p, n, None) == 1 and call(eng.plan, ws, 0, p + 4, n, None) == 1
        assert call(eng.plan, ws, 0, p, n - 1, None) == 1 and call(eng.plan, ws, 0, None, n, None) == 1
    ev = m.eval().engine_for(x)
    assert lib.csn_plan_checkpoint_bytes(ev.plan) == 0
    with pytest.raises(ValueError):
        m.set_train_checkpoints("fp4")


def test_views_of_slices():
    """Every slice, permutation and broadcast that is read as it lies, or copied, has the elements of the tensor in its order."""
    from sod100k_amd.train_ops import _view
    base = torch.arange(4 * 6 * 3 * 5).reshape(4, 6, 3, 5)
    cuts = (slice(None), slice(1, None), slice(0, 1), slice(None, None, 2))
    as_it_lies = 0
    for perm in ((0, 1, 2, 3), (1, 0, 2, 3), (0, 2, 3, 1), (3, 2, 1, 0)):
        for cut in ((a, b, c, d) for a in cuts for b in cuts for c in cuts for d in cuts):
            x = base.permute(perm)[cut]
            for t in (x, x[:, :, :1].expand(-1, -1, 3, -1), x[:1].expand(2, -1, -1, -1), x[0], x[0, 0]):
                for rows in (True, False) if t.dim() > 2 else (True,):
                    v, so, sc = _view(t, rows)
                    want = t.reshape(-1, t.shape[-1]) if rows else t.flatten(2)
                    got = torch.as_strided(v, want.shape, (so, 1) if rows else (so, sc, 1), v.storage_offset())
                    assert torch.equal(got, want)
                    as_it_lies += v.data_ptr() == t.data_ptr()
    assert as_it_lies > 1000
    x = torch.zeros(4, 10, 6, 7)
    for t, rows in ((x[:, 2:9], False), (x[1:], False), (x.reshape(-1, 7)[:, 1:5], True), (x[..., 2:], True)):
        assert _view(t, rows)[0].data_ptr() == t.data_ptr()      # slices of channels and images are not copied
