"""Whole models of the designs that hold some matrices in 8 bits among other parts, against the same models on the bfloat16 path with what 8 bits stand for: the
matrices replaced by the numbers of their codes and powers (which bfloat16 holds exactly), their rows brought to 8 bits before a plain float32 product.

Both engines round to bfloat16 around these products, in other places: the rows before 8 bits (a norm hands them on without), the products' results (float32 sums
for some consumers).  Such a rounding is half a step, 2^-8 of a value, at most, and where it carries a value over a border between two e4m3 numbers, a step of those.  How far
that moves a model's logits is measured on the reference alone: rows and results moved by random shares of half a step.  The bound is twice the largest
distance of three such runs: what separates the engines is as much again, at other borders."""
import contextlib
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
K = importlib.import_module("daisi-llogos_amd.ops.kernels")
base = importlib.import_module("daisi-llogos_amd.parts.base")
linear = importlib.import_module("daisi-llogos_amd.parts.linear")
Linear = linear.Linear
BF16 = torch.bfloat16
SEQS, PROMPT, STEPS = 2, 20, 4


class Reference:
    """Linear's methods for a matrix that would be held in 8 bits; moved: a generator whose random shares of half a bfloat16 step rows and results are moved by."""

    def __init__(self):
        self.moved = None
        self.saved = {n: getattr(Linear, n) for n in ("bind", "product", "gated_product", "add_to", "forward")}

    def _move(self, v):
        return v if self.moved is None else v * (1 + 2.0 ** -8 * (2 * torch.rand(v.shape, generator=self.moved, device=v.device) - 1))

    def _whole(self, lin, a):
        a = a.tensor() if isinstance(a, base.NormedRows) else a
        rows = K.quantize_rows(self._move(a.float())).values()
        return rows @ lin.weight.float().t()

    def _done(self, v):
        return self._move(v).to(BF16)

    @contextlib.contextmanager
    def patched(self):
        saved, ref = self.saved, self

        def bind(lin, get, rt):
            saved["bind"](lin, get, rt)
            if lin.eight_bit:
                stored = linear._to_device([get(n + lin.suffix) for n in lin.names], torch.float32, rt.device)
                codes, powers = K.quantize_weight(stored)
                of = powers.float().repeat_interleave(128, 0)[:stored.shape[0]].repeat_interleave(128, 1)[:, :stored.shape[1]]
                lin.weight, lin.packed = (codes.float() * of).to(BF16), None
                assert torch.equal(lin.weight.float(), codes.float() * of)

        def product(lin, a, rows_out=None, swiglu_input=False, f32_ok=False):
            if not lin.eight_bit:
                return saved["product"](lin, a, rows_out, swiglu_input, f32_ok)
            if swiglu_input:
                half = a.shape[-1] // 2
                a = (torch.nn.functional.silu(a[..., :half].float()) * a[..., half:].float())
            return ref._done(ref._whole(lin, a))[:, :rows_out].contiguous()

        def gated_product(lin, a, limit=None, block_rows=False):
            if not lin.eight_bit:
                return saved["gated_product"](lin, a, limit, block_rows)
            gu = ref._whole(lin, a)
            half = gu.shape[-1] // 2
            return ref._done(torch.nn.functional.silu(gu[:, :half]) * gu[:, half:])

        def add_to(lin, a, residual):
            return None if lin.eight_bit else saved["add_to"](lin, a, residual)

        def forward(lin, a, out_dtype=None, rows_out=None):
            assert not lin.eight_bit
            return saved["forward"](lin, a, out_dtype, rows_out)
        with pytest.MonkeyPatch.context() as mp:
            for n, f in (("bind", bind), ("product", product), ("gated_product", gated_product), ("add_to", add_to), ("forward", forward)):
                mp.setattr(Linear, n, f)
            yield


def logits(eng, toks):
    """Of every position: the prompts' in one step, then single tokens."""
    slots = [eng.alloc_slot() for _ in toks]
    rows = [eng.step([(s, t[:PROMPT]) for s, t in zip(slots, toks)], "all").double().cpu()]
    for i in range(PROMPT, PROMPT + STEPS):
        rows.append(eng.step([(s, [t[i]]) for s, t in zip(slots, toks)], "last").double().cpu())
    for s in slots:
        eng.free_slot(s)
    out = torch.cat(rows).numpy()
    assert np.isfinite(out).all()
    return out - out.mean(axis=1, keepdims=True)          # (what all logits of a position share says nothing)


def apart(a, b):
    """The largest distance of a position's logits, of their size."""
    return (np.linalg.norm(a - b, axis=1) / np.linalg.norm(b, axis=1)).max()


DESIGNS = [("batodra", n) for n in ("bat_a", "bat_b", "bat_c")] + [("zasidra", n) for n in ("zas_a", "zas_b", "zas_c", "zas_d")] + \
    [("peponex", n) for n in ("pep_a", "pep_b", "pep_c", "pep_e")] + [("zisedra", n) for n in ("zis_a", "zis_b", "zis_c", "zis_d", "zis_e")]


@pytest.mark.parametrize("design,name", DESIGNS)
def test_designs_in_8_bits(design, name):
    helpers = importlib.import_module(design + "_helpers")
    eight = helpers.engine(name, "bfloat16", weights="fp8")
    rng = np.random.default_rng(11)
    toks = rng.integers(0, eight.vocab_size, size=(SEQS, PROMPT + STEPS)).tolist()
    got = logits(eight, toks)
    ref = Reference()
    with ref.patched():
        eng = helpers.engine(name, "bfloat16", use_graphs=False)
        want = logits(eng, toks)
        far = []
        for seed in range(3):
            ref.moved = torch.Generator(device="cuda").manual_seed(seed)
            far.append(apart(logits(eng, toks), want))
    bound = 2 * max(far)
    off = apart(got, want)
    print(f"{name}: {off:.4f} apart, bound {bound:.4f}, from bfloat16 matrices {apart(logits(helpers.engine(name, 'bfloat16'), toks), want):.4f}")
    assert off <= bound
