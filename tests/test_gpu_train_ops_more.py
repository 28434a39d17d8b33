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
