"""Powers of two at the ends of their byte, in rows and matrices that a caller brings (block_rows, block_weight): every byte is a power 2^(byte - 127), 255 is NaN."""
import importlib

import numpy as np
import pytest
import torch

import plain_blocks8 as p8

pytestmark = pytest.mark.gpu
K = importlib.import_module("daisi-llogos_amd.ops.kernels")
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
FORMS = [0, 1, 10401, 10801, 11201, 11601, 20401, 40403]
M, N, KK = 37, 160, 384


def _operands(seed, ea, ew, small=False):
    """Codes of all sizes (small: the eight smallest), the bytes of the rows' powers [M, 3] and of the matrix's [2, 3]."""
    rng = np.random.default_rng(seed)
    a, w = (rng.integers(0, 8 if small else 127, size=s) | (rng.integers(0, 2, size=s) << 7) for s in ((M, KK), (N, KK)))
    dev = lambda v, t: torch.tensor(np.asarray(v).astype(np.uint8), device="cuda").view(t)  # noqa: E731
    ea, ew = np.broadcast_to(ea, (M, 3)), np.broadcast_to(ew, (2, 3))
    return K.block_rows(dev(a, E4M3), dev(ea, E8M0)), K.block_weight(dev(w, E4M3), dev(ew, E8M0)), p8.values(a, ea.astype(int) - 127), p8.values(w, ew.astype(int) - 127, 128)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("ea,ew,small", [(254, 0, False), (0, 254, False), (254, 10, False), (20, 230, False), (1, 240, False), (200, 160, True), (230, 130, True)])
def test_powers_far_apart(form, ea, ew, small):
    """One side's as large as the other's are small, and sums of exponents beyond float32's with codes that bring the products back.  (The bound of the
    products: 2^-12 of the products' sizes and a rounding to bfloat16.)"""
    rows, weight, a, w = _operands(ea + ew, ea, ew, small)
    want, size = a @ w.T, np.abs(a) @ np.abs(w).T
    assert 1e-30 < np.abs(want).max() < 2.0 ** 127
    got = K.gemm_blocks(rows, weight, form=form).double().cpu().numpy()
    off = 2.0 ** -12 * size
    assert (np.abs(got - want) <= off + 2.0 ** -8 * (np.abs(want) + off)).all()


@pytest.mark.parametrize("form", FORMS)
def test_a_power_that_is_no_number(form):
    ea, ew = np.full((M, 3), 127), np.full((2, 3), 120)
    ea[5, 1], ew[1, 2] = 255, 255
    rows, weight, a, w = _operands(7, ea, ew)
    assert torch.isnan(rows.values()[5, 128:256]).all()
    got = K.gemm_blocks(rows, weight, form=form).double().cpu().numpy()
    bad = np.zeros((M, N), dtype=bool)
    bad[5], bad[:, 128:] = True, True
    assert np.array_equal(np.isnan(got), bad)
