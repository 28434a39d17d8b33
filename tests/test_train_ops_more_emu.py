"""Further checks of the training operators beside the plan on the CPU emulation of their kernels (lane-exact mode)."""
import pytest
import torch

import train_ops_cases as K
import train_ops_more as M


@pytest.fixture(scope="module")
def lib(emu_lanes_lib):
    return emu_lanes_lib[0]


@pytest.mark.parametrize("dtype", K.DTYPES)
@pytest.mark.parametrize("shape,dim", M.CONSTANT)
def test_emu_constant_tokens(lib, shape, dim, dtype):
    M.check_constant_tokens(lib, "cpu", shape, dim, dtype)


@pytest.mark.parametrize("shape,dim", [((3, 100), -1), ((2, 40, 3, 5), 1)])
def test_emu_nan_statistics(lib, shape, dim):
    M.check_nan_statistics(lib, "cpu", shape, dim)


def test_emu_without_gradients(lib, monkeypatch):
    M.check_without_gradients(lib, "cpu", monkeypatch)


def test_emu_frozen_norm(lib, monkeypatch):
    M.check_frozen_norm(lib, "cpu", monkeypatch)


def test_emu_autocast(lib):
    M.check_autocast(lib, "cpu")


def test_refusals_of_workspaces(lib):
    M.check_refusals_of_workspaces(lib)


def test_refusals_of_workspaces_of_the_product_library():
    import ctypes
    import os
    from sod100k_amd import _native as N
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("libcsnet_hip.so not built")
    M.check_refusals_of_workspaces(N.bind(ctypes.CDLL(N.LIB_PATH)))


def test_emu_outputs_end_where_they_end(lib):
    M.check_outputs_end_where_they_end(lib, "cpu")
