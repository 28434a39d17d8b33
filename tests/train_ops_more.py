"""Further checks of the training operators beside the plan, shared by the emulator suite (tests/test_train_ops_more_emu.py) and the GPU
suite (tests/test_gpu_train_ops_more.py).  Oracles and tolerances: train_ops_cases.py."""
import pytest
import torch

import train_ops_cases as K
from sod100k_amd import _native as N, train_ops as T

# tokens whose channels are all the same number, which a float sum of so many does not give back
CONSTANT = [(shape, dim) for ch in (331, 1000, 2048) for shape, dim in (((3, ch), -1), ((2, ch, 3, 5), 1))] + [((2, 9000), -1)]


def check_constant_tokens(lib, dev, shape, dim, dtype):
    """The mean is that number, the normalised value zero and rstd that of no variance at all: x - m for m near x is exact, so are the
    sums of C equal small multiples of a last place, and their quotient."""
    w, b = K.params(shape[dim], 8, dev)
    for v in (0.1, 1000.1, 30000.7, -3.0e7):
        x = torch.full(shape, v, dtype=torch.float64).to(dtype).to(dev)
        y, mean, rstd, _ = T.layer_norm_forward(lib, x, w, b, dim=dim)
        want = (b if dim == -1 else b.view(1, -1, 1, 1)).expand(shape)
        assert torch.equal(y, want.to(dtype)), v
        assert bool((mean == x.select(dim, 0).float()).all()), v
        assert bool(((rstd.cpu().double() - 1e5 ** 0.5).abs() <= 4 * K.U * 1e5 ** 0.5).all()), v


def check_nan_statistics(lib, dev, shape, dim):
    """A NaN or an infinity in a token leaves no number in its mean and rstd."""
    x = K.activations(shape, torch.float32, 3, dev, rows=dim == -1)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z.select(dim, 1).fill_(bad)
        _, mean, rstd, _ = T.layer_norm_forward(lib, z, dim=dim)
        assert not bool(torch.isfinite(mean).any()) and bool(torch.isnan(rstd).all())
