"""The 8-bit product at the ends of its arrays: tiles of 192 tokens, whose lanes read the powers of 12 tokens at once, where those lie across the last byte of the powers."""
import importlib

import numpy as np
import pytest

import plain_blocks8 as p8
from test_blocks8_gpu import K, _bits, _np, _product_case, E4M3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [13, 16, 25, 30, 31, 32, 205, 208, 222, 224, 398, 400])
@pytest.mark.parametrize("k", [128, 640])
def test_powers_of_twelve_tokens_across_the_end(M, k):
    """(16 ceil(M / 16) bytes a block of k: the last ones are no multiple of 12 behind a tile's first)"""
    rows, weight, b, want, off = _product_case(M, 80, k, bias=True)
    got = K.gemm_blocks(rows, weight, b, form=11201)
    over = np.abs(_np(got) - want) - off
    assert over.max() <= 0, f"{(over > 0).sum()} of {over.size} values beyond their tolerance, rows {sorted(set(np.argwhere(over > 0)[:, 0].tolist()))}"


@pytest.mark.parametrize("M", [30, 208, 222])
def test_gated_rows_of_twelve_tokens_across_the_end(M):
    rows, weight, _, want, off = _product_case(M, 80, 640, gated=True, spread=2)
    got = K.gemm_blocks(rows, weight, form=11201, out_dtype=E4M3)
    e = _bits(got.powers) - 127
    v, p = p8.values(_bits(got.codes), e), np.repeat(2.0 ** e.astype(np.float64), 128, axis=1)[:, :80]
    over = np.abs(v - want) - off - np.maximum(2.0 ** -4 * (np.abs(want) + off), 2.0 ** -10 * p)
    assert over.max() <= 0, f"{(over > 0).sum()} of {over.size} values beyond their tolerance"
