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
