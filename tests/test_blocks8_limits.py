"""What the 8-bit operators refuse because the kernels count in 32 bits.  Tensors without memory ("meta") stand for the large ones: a call ends before it looks for a GPU."""
import importlib

import pytest
import torch

K = importlib.import_module("daisi-llogos_amd.ops.kernels")
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BF16 = torch.bfloat16
FAR = 2 ** 31


def m(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("call", [
    lambda: K.quantize_rows(m(FAR + 5, 8)),
    lambda: K.quantize_rows(m(2, FAR + 3, 8)),
    lambda: K.quantize_rows(m(1, FAR + 128, dtype=BF16)),
    lambda: K.quantize_rows(m(1, 2 * FAR + 256, dtype=BF16), gated=True),
    lambda: K.quantize_rows(m(FAR + 5, 2, 8)),
    lambda: K.quantize_weight(m(FAR + 1, 1)),
    lambda: K.quantize_weight(m(1, FAR + 1)),
    lambda: K.block_rows(m(FAR + 1, 1, dtype=E4M3), m(FAR + 1, 1, dtype=E8M0)),
    lambda: K.block_rows(m(1, FAR, dtype=E4M3), m(1, FAR // 128, dtype=E8M0)),
    lambda: K.block_weight(m(FAR, 1, dtype=E4M3), m(FAR // 128, 1, dtype=E8M0)),
    lambda: K.block_weight(m(1, FAR, dtype=E4M3), m(1, FAR // 128, dtype=E8M0)),
    lambda: K.gated_norms(m(FAR + 5, 1), None, 1e-5, alpha=0.5),
    lambda: K.gated_norms(m(3, 8), m(FAR + 1, 3, 8), 1e-5),
])
def test_sizes_beyond_32_bits(call):
    with pytest.raises(K.KernelError, match="2\\^31"):
        call()


@pytest.mark.parametrize("form", [-1, -10401, FAR + 1, 2 * FAR + 1, 2 * FAR + 10416])
@pytest.mark.parametrize("rows", [lambda: K.BlockRows(3, 256, torch.empty(0)), lambda: torch.zeros(3, 256, dtype=BF16), lambda: torch.zeros(40, 256, dtype=BF16)])
def test_forms_that_are_none(form, rows):
    """(as a C int 2^32 + 10,416 would be 16 parts, with room for 12 of them)"""
    w = K.BlockWeight(torch.zeros(64 * 128, dtype=BF16), torch.ones(1, 2, 4, dtype=torch.uint8), 64, 256)
    with pytest.raises(K.KernelError, match="form"):
        K.gemm_blocks(rows(), w, form=form)
