"""Forwards that wait for their backward (CSNet.set_train_checkpoints) on the CPU emulation of the kernels."""
import pytest
import torch

import waiting_cases as W

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def lib(emu_lanes_lib):
    return emu_lanes_lib[0]


@pytest.mark.parametrize("act_dtype", ["fp32", "bf16"])
def test_emu_refilled_batch(lib, x2_manifest, act_dtype):
    W.check_refilled_batch(lib, CPU, x2_manifest, act_dtype)
