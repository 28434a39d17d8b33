"""Forwards that wait for their backward (CSNet.set_train_checkpoints) on the GPU."""
import pytest
import torch

import waiting_cases as W
from sod100k_amd import _native as N

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.fail("the GPU suite needs a ROCm device")
    return N.load()


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
def test_gpu_refilled_batch(lib, x2_manifest, act_dtype):
    W.check_refilled_batch(lib, DEV, x2_manifest, act_dtype)


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
def test_gpu_two_streams(lib, x2_manifest, act_dtype):
    W.check_two_streams(lib, DEV, x2_manifest, act_dtype, B=8, size=96, rounds=3)


def test_gpu_changed_parameters(lib, x2_manifest):
    W.check_changed_parameters(lib, DEV, x2_manifest)


def test_gpu_failed_save(lib, x2_manifest):
    W.check_failed_save(lib, DEV, x2_manifest)


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
def test_gpu_penalty_and_input_gradients(lib, x2_manifest, act_dtype):
    W.check_penalty_and_input_gradients(lib, DEV, x2_manifest, act_dtype, B=3, size=48)


def test_gpu_failed_forward(lib, x2_manifest):
    W.check_failed_forward(lib, DEV, x2_manifest)
