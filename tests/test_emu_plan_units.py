"""The emulator built from the plan's units alone, without the training operators' kernels: it loads, the network runs on it, and the
operators that it lacks are refused."""
import ctypes as C
import os
import subprocess

import torch

import emu_build
import parity_cases as P
from oracle import inputs as I
from sod100k_amd import _native as N, train_ops as T

OPERATORS = ("k_q8.hip", "k_norm.hip", "k_q8_wgrad.hip")


def test_plan_units_alone(emu_lanes_lib, x2_manifest, tmp_path):
    so = str(tmp_path / "libcsnet_emu_plan.so")
    srcs = " ".join("../../sod100k_amd/csrc/" + s for s in N.SOURCES if s not in OPERATORS)
    subprocess.run(["make", "-C", emu_build.EMU, "-j8", "LANES=1", "OUT=" + so, "SRCS=" + srcs], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.PIPE)
    assert os.path.exists(so)
    lib = N.bind(C.CDLL(so))
    x = torch.from_numpy(I.randn_batch(5, 1, 32, 32))
    out = []
    for b in (lib, emu_lanes_lib[0]):
        m, _ = P.make_model(b, x2_manifest, torch.device("cpu"))
        with torch.no_grad():
            out.append(m.eval()(x))
    assert torch.equal(*out)

    p = C.c_void_p(4096)      # never followed
    d = N.NormDesc(N.LAYOUT_ROWS, N.DTYPE_F32, 4, 8, 1, 1e-5, 0)
    w = N.ProductDesc(N.LAYOUT_ROWS, N.DTYPE_F32, 0, 0, 4, 1, 8, 8)
    big = 1 << 40
    for status in (lib.csn_q8_pack(p, 0, 1, 4, 4, 0, 4, 0, p, p, None), lib.csn_q8_unpack(p, p, 0, 4, 4, p, 0, None),
                   lib.csn_layer_norm_forward(C.byref(d), p, 8, 0, None, None, p, None, None, None, None, None),
                   lib.csn_layer_norm_backward(C.byref(d), p, 8, 0, p, 8, 0, None, None, p, p, None, p, p, p, p, big, None),
                   lib.csn_product_weight_grad(C.byref(w), p, 8, 0, p, p, p, None, p, big, None),
                   lib.csn_plan_checkpoint_save(p, p, 0, p, big, None), lib.csn_plan_checkpoint_restore(p, p, 0, p, big, None)):
        assert status == 2 and b"without" in lib.csn_last_hip_error()
    assert lib.csn_layer_norm_workspace_bytes(C.byref(d)) == 0 and lib.csn_product_weight_grad_workspace_bytes(C.byref(w)) == 0
    try:
        T.q8_pack(lib, torch.zeros(2, 4))
    except RuntimeError as e:
        assert "without" in str(e)
    else:
        raise AssertionError("packed without a kernel")
