"""Training operators beside the plan on the GPU: the emulator suite's checks at its and at larger sizes, captured, on other streams
and next to each other."""
import pytest
import torch

import train_ops_cases as K
from sod100k_amd import _native as N, train_ops as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.fail("the GPU suite needs a ROCm device")
    return N.load()


DEV = "cuda:0"


@pytest.mark.parametrize("fmt", K.FORMATS)
@pytest.mark.parametrize("dtype", K.DTYPES)
def test_gpu_pack(lib, fmt, dtype):
    for i, (shape, start) in enumerate(K.PACK_SHAPES + [((3, 1000), -1), ((2, 5, 33, 31), 2)]):
        K.check_pack(lib, K.activations(shape, dtype, i, DEV, rows=start == -1), fmt, start)
    K.check_pack(lib, K.block_edge_values(dtype).to(DEV), fmt, -1)


@pytest.mark.parametrize("fmt", K.FORMATS)
def test_gpu_every_code(lib, fmt):
    q, want = K.every_code_once(fmt, DEV)
    for dtype in K.DTYPES:
        assert K.same(T.q8_unpack(lib, q, dtype).cpu().double(), want)


@pytest.mark.parametrize("fmt", K.FORMATS)
def test_gpu_every_bfloat16(lib, fmt):
    """All 65536 bfloat16 numbers, each in a block of its own magnitude and all in mixed blocks: the rounding of the codes."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    K.check_pack(lib, bits.view(2048, 32).to(DEV), fmt, -1)
    mixed = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(0))].view(2048, 32)
    K.check_pack(lib, mixed.to(DEV), fmt, -1)


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape,dim", K.NORM_SHAPES + [((3000, 256), -1), ((4, 40, 56, 56), 1), ((2, 256, 22, 22), 1), ((600, 2048), -1),
                                                       ((3, 80, 111, 37), 1), ((1, 2048, 11, 11), 1)])
def test_gpu_norm(lib, shape, dim, dtype):
    rows = dim == -1
    x, dy = K.activations(shape, dtype, 1, DEV, rows=rows), K.gradient(shape, dtype, 1, DEV)
    w, b = K.params(shape[dim], 1, DEV)
    big = x.numel() > 100000      # (the checkpoint's oracle walks every block in Python)
    y, mean, rstd, _ = K.check_norm_forward(lib, x, w, b, dim)
    K.check_norm_forward(lib, x, None, None, dim)
    K.check_norm_backward(lib, dy, x, mean, rstd, w, dim)
    K.check_norm_backward(lib, dy, x, mean, rstd, None, dim)
    for fmt in K.FORMATS:
        if big:
            y2, m2, r2, q = T.layer_norm_forward(lib, x, w, b, dim=dim, checkpoint=fmt)
            p = T.q8_pack(lib, x, fmt, start_dim=-1 if rows else 2)
            assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
            dq = T.layer_norm_backward(lib, dy, q, mean, rstd, w, dim=dim)
            ref = T.layer_norm_backward(lib, dy.float(), T.q8_unpack(lib, q), mean, rstd, w, dim=dim)
            assert torch.allclose(dq[0].float(), ref[0], rtol=2 * K.HALF[dtype], atol=64 * K.U * float(ref[0].abs().max()))
            for s, t in zip(dq[1:], ref[1:]):
                assert torch.allclose(s, t, rtol=0, atol=2048 * K.U * float(dy.abs().float().sum()) / shape[dim] * 8)
        else:
            y2, m2, r2, q = K.check_norm_forward(lib, x, w, b, dim, checkpoint=fmt)
            K.check_norm_backward(lib, dy, x, mean, rstd, w, dim, q=q)
        assert torch.equal(y, y2) and torch.equal(mean, m2) and torch.equal(rstd, r2)


@pytest.mark.parametrize("fmt", K.FORMATS)
@pytest.mark.parametrize("dtype", K.DTYPES)
def test_gpu_product_gradient(lib, dtype, fmt):
    for i, (dims, cin, cout, dim) in enumerate(K.PRODUCT_SHAPES + [((513,), 300, 280, -1), ((2, 31, 33), 129, 257, 1), ((3, 24, 24), 256, 128, 1),
                                                                   ((1030,), 128, 512, -1), ((2051,), 500, 1200, -1), ((70000,), 264, 257, -1)]):
        x, dy = K.product_tensors(dims, cin, cout, dim, dtype, i, DEV)
        K.check_product(lib, dy, x, fmt, dim)


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_gpu_slices_and_strides(lib, dtype):
    K.check_slices(lib, DEV, dtype)


def test_gpu_empty(lib):
    K.check_empty(lib, DEV)


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_gpu_bad_tokens_stay_alone(lib, dtype):
    K.check_bad_tokens_stay_alone(lib, DEV, dtype)


def test_gpu_constant_tokens_and_far_means(lib):
    K.check_constant_and_far(lib, DEV)


def test_gpu_determinism(lib):
    K.check_determinism(lib, DEV)


def test_gpu_gradients_against_differences(lib):
    K.check_against_differences(lib, DEV)


@pytest.mark.parametrize("dtype", K.DTYPES)
def test_gpu_norm_and_product_together(lib, dtype):
    K.check_block_of_operators(lib, DEV, dtype)


def test_gpu_refusals(lib):
    K.check_refusals(lib, DEV)
    with pytest.raises(RuntimeError, match="ROCm"):
        T.q8_pack(lib, torch.zeros(2, 4))


def test_gpu_captured_and_replayed(lib):
    """Two graphs captured one after the other, replayed in turn with eager work between: every replay gives the eager results."""
    sets = []
    for seed in (1, 2):
        x, dy = K.activations((2, 40, 30, 31), torch.bfloat16, seed, DEV, rows=False), K.gradient((2, 40, 30, 31), torch.bfloat16, seed, DEV)
        w, b = K.params(40, seed, DEV)
        sets.append((x, dy, w, b))
    want = [K._all_of(T, lib, *s, 1) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K._all_of(T, lib, *s, 1))
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1):
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
            K._all_of(T, lib, *sets[1 - i], 1)        # eager work with the other set
            torch.cuda.synchronize()
            for o, v in zip(outs[i], want[i]):
                assert torch.equal(o, v)


def test_gpu_gradients_refuse_a_capture(lib):
    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            T.layer_norm(x)
        torch.zeros(1, device=DEV)
    with torch.no_grad():
        T.layer_norm(x)


def test_gpu_other_streams(lib):
    """The same operators on several streams at once: each call has a workspace of its own."""
    sets = []
    for seed in range(4):
        x, dy = K.activations((3, 64, 40, 41), torch.float32, seed, DEV, rows=False), K.gradient((3, 64, 40, 41), torch.float32, seed, DEV)
        sets.append((x, dy, *K.params(64, seed, DEV)))
    want = [K._all_of(T, lib, *s, 1) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(K._all_of(T, lib, *s, 1))
        torch.cuda.synchronize()
        for g, v in zip(got, want):
            for a, b in zip(g, v):
                assert torch.equal(a, b)


def test_gpu_outputs_end_where_they_end(lib):
    """Memory behind every output stays as it was (odd sizes, vectors that would run past the end)."""
    import ctypes as C
    for dtype, dt in ((torch.float32, 0), (torch.bfloat16, 1)):
        for rows, shape in ((True, (5, 33)), (True, (3, 256)), (False, (2, 7, 35)), (False, (1, 12, 64))):
            x, dy = K.activations(shape, dtype, 1, DEV, rows=rows), K.gradient(shape, dtype, 1, DEV)
            o, c, p = (shape[0], shape[1], 1) if rows else shape
            n, tok = x.numel(), o * p
            nsc = o * (-(-c // 32)) if rows else o * c * (-(-p // 32))
            pad = 64

            def buf(k, t):
                return torch.full((k + pad,), 77, dtype=t, device=DEV)
            y, codes, sc, mean, rstd, dx = buf(n, dtype), buf(n, torch.uint8), buf(nsc, torch.uint8), buf(tok, torch.float32), buf(tok, torch.float32), buf(n, dtype)
            dw, db, val = buf(c, torch.float32), buf(c, torch.float32), buf(n, dtype)
            d = N.NormDesc()
            d.layout, d.dtype, d.outer, d.channels, d.inner, d.eps, d.format = int(rows), dt, o, c, p, 1e-5, 0
            so, scs = (c, 0) if rows else (c * p, p)
            st = torch.cuda.current_stream().cuda_stream
            N.check(lib, lib.csn_layer_norm_forward(C.byref(d), x.data_ptr(), so, scs, None, None, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                                    codes.data_ptr(), sc.data_ptr(), st), "fwd")
            nb = lib.csn_layer_norm_workspace_bytes(C.byref(d))
            ws = buf(nb, torch.uint8)
            N.check(lib, lib.csn_layer_norm_backward(C.byref(d), dy.data_ptr(), so, scs, None, 0, 0, codes.data_ptr(), sc.data_ptr(), mean.data_ptr(),
                                                     rstd.data_ptr(), None, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nb, st), "bwd")
            N.check(lib, lib.csn_q8_unpack(codes.data_ptr(), sc.data_ptr(), 0, o if rows else o * c, c if rows else p, val.data_ptr(), dt, st), "unpack")
            for t, k in ((y, n), (codes, n), (sc, nsc), (mean, tok), (rstd, tok), (dx, n), (dw, c), (db, c), (val, n), (ws, nb)):
                assert bool((t[k:] == 77).all())


def test_gpu_offsets_beyond_32_bits(lib):
    """Tensors of more than 2^31 elements: the last tokens' results are those of the tail alone."""
    n, c = (1 << 31) // 1024 + 3, 1024
    x = torch.empty((n, c), dtype=torch.bfloat16, device=DEV)
    tail = K.activations((6, c), torch.bfloat16, 1, DEV)
    x.zero_()
    x[-6:] = tail
    q = T.q8_pack(lib, x, "int8")
    qt = T.q8_pack(lib, tail, "int8")
    assert torch.equal(q.codes[-6:], qt.codes) and torch.equal(q.scales[-6:], qt.scales) and not bool(q.codes[:-6].any())
    v = T.q8_unpack(lib, q, torch.bfloat16)
    assert torch.equal(v[-6:], T.q8_unpack(lib, qt, torch.bfloat16))
    del v
    y, mean, rstd, _ = T.layer_norm_forward(lib, x)
    yt, mt, rt, _ = T.layer_norm_forward(lib, tail)
    assert torch.equal(y[-6:], yt) and torch.equal(mean[-6:], mt) and torch.equal(rstd[-6:], rt)
    dyt = K.gradient((6, c), torch.bfloat16, 1, DEV)
    y.zero_()
    y[-6:] = dyt
    dx, dw, db = T.layer_norm_backward(lib, y, x, mean, rstd)
    dxt, dwt, dbt = T.layer_norm_backward(lib, dyt, tail, mt, rt)
    assert torch.equal(dx[-6:], dxt)
    assert torch.allclose(dw, dwt, rtol=1e-5, atol=1e-6) and torch.allclose(db, dbt, rtol=1e-5, atol=1e-6)
    del dx
    dW, dB = T.product_weight_grad(lib, y[:, :8], q)
    ref, _ = T.product_weight_grad(lib, dyt[:, :8], qt)
    assert torch.allclose(dW, ref, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("fmt", K.FORMATS)
def test_gpu_plan_checkpoint(lib, x2_manifest, act_dtype, fmt):
    K.check_plan_checkpoint(lib, torch.device(DEV), x2_manifest, act_dtype, fmt, B=3, size=64)


@pytest.mark.parametrize("act_dtype,fmt", [("fp32", "e4m3"), ("bf16", "int8")])
def test_gpu_two_forwards_one_backward(lib, x2_manifest, act_dtype, fmt):
    K.check_two_forwards_one_backward(lib, torch.device(DEV), x2_manifest, act_dtype, fmt, B=2, size=48)


def test_gpu_waiting_forwards_refuse(lib, x2_manifest):
    K.check_waiting_forwards_refuse(lib, torch.device(DEV), x2_manifest, B=2, size=48)
