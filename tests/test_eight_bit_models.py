"""Models under weights='fp8' without a GPU: which are refused, and what memory their matrices are counted on to take."""
import contextlib
import importlib

import pytest
import torch

import nipulorn_configs
import peponex_configs
import tiny_configs
import zasidra_configs
import zogurax_configs

K = importlib.import_module("daisi-llogos_amd.ops.kernels")
L = importlib.import_module("daisi-llogos_amd")
base = importlib.import_module("daisi-llogos_amd.parts.base")
reg = importlib.import_module("daisi-llogos_amd.config.registry")
step = importlib.import_module("daisi-llogos_amd.engine.step")


def model_of(config):
    arch = reg.architecture_of(config)
    return L.Model(arch.model_spec(arch.read_config(config)))


WITHOUT = {**nipulorn_configs.ALL, **zogurax_configs.ALL, "pep_d": peponex_configs.PEP_D}       # (no attention or SwiGLU of the kinds that go in 8 bits)
WITH = {"tiny_a": tiny_configs.TINY_A, "zas_a": zasidra_configs.ZAS_A, "pep_a": peponex_configs.PEP_A}


@pytest.mark.parametrize("name", sorted(WITHOUT))
def test_models_without_such_matrices_are_refused(name):
    model = model_of(WITHOUT[name])
    assert model.eight_bit_matrices() == 0
    with pytest.raises(ValueError, match="no matrix that can be held in fp8"):
        step._needs_eight_bit(model)


@pytest.mark.parametrize("name", sorted(WITH))
def test_models_with_such_matrices_are_not(name):
    model = model_of(WITH[name])
    assert model.eight_bit_matrices() > 0
    step._needs_eight_bit(model)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["nip_a", "zog_a"])
def test_an_engine_refuses_them(name):
    with pytest.raises(ValueError, match="no matrix that can be held in fp8"):
        L.Engine.from_config(WITHOUT[name], weights="fp8")


def linears(part, found=None):
    """All products of a part and its sub-parts."""
    found = [] if found is None else found
    for v in vars(part).values():
        for x in v if isinstance(v, (list, tuple)) else [v]:
            if isinstance(x, base.Part):
                if type(x).__name__ == "Linear":
                    found.append(x)
                linears(x, found)
    return found


def bound8(monkeypatch, config, free):
    """The model of `config` bound in 8 bits on the CPU, with copies made by ordinary tensors of their sizes; free: bytes for copies beside matrices and cache (None:
    as packed_weight_budget says)."""
    monkeypatch.setattr(K, "pack_weights", lambda w, gate_rows=0: K.PackedWeight(
        torch.zeros(K.packed_weight_bytes(*w.shape) // 2, dtype=torch.bfloat16), *w.shape, gate_rows))
    monkeypatch.setattr(K, "quantize_weight", lambda w: (w, None))

    def block(w, _, gate_rows=0, **more):
        blocks = -(-w.shape[1] // 128)
        rows = -(-w.shape[0] // 64)
        return K.BlockWeight(torch.zeros(rows * 64 * blocks * 64, dtype=torch.bfloat16), torch.zeros(rows, blocks, 4, dtype=torch.uint8), *w.shape, gate_rows)
    monkeypatch.setattr(K, "block_weight", block)
    model = model_of(config)
    rt = base.Runtime(torch.device("cpu"), torch.bfloat16, eight_bit=True)
    if free is not None:
        monkeypatch.setattr(step, "packed_weight_budget", lambda *a: free)
    step._packing(rt, model, 64, None)
    shapes = {s.name: s for s in model.tensor_specs()}
    model.bind(lambda name: torch.zeros(shapes[name].shape) if name in shapes else None, rt)
    return model, rt


def experts_of(model):
    return [w for layer in model.layers for f in layer.feed_forwards() if hasattr(f, "packed_up") for w in (f.packed_up, f.packed_down)]


@pytest.mark.parametrize("config", [zasidra_configs.ZAS_C, peponex_configs.PEP_C])
def test_matrices_in_8_bits_are_no_copies_to_make_room_for(monkeypatch, config):
    """Experts get what the copies that are made, and a second engine like this one, leave: a matrix in 8 bits has no copy and takes a byte an element."""
    model, rt = bound8(monkeypatch, config, 1 << 40)
    experts = [e for e in experts_of(model) if e is not None]            # (those whose sizes have a packed form)
    in_8_bits = [l for layer in model.layers for l in linears(layer) if l.block is not None]
    assert len(in_8_bits) == model.eight_bit_matrices() and experts
    each = sum(e.data.numel() * 2 for e in experts)
    others = model.packed_weight_bytes() - each
    assert model.packable_bytes(True) == others == model.packable_bytes() - sum(K.packed_weight_bytes(l.total_out, l.in_features) for l in in_8_bits)
    new = model_of(config)                                              # (counted before it is bound)
    native, own = step._own_bytes(new, torch.bfloat16, 64), step._own_bytes(new, torch.bfloat16, 64, True)
    assert own == native - 2 * sum(l.matrix_elements() for l in in_8_bits) + sum(l.block.bytes() for l in in_8_bits)
    model, rt = bound8(monkeypatch, config, 2 * others + own + each)
    assert sum(e is not None for e in experts_of(model)) == len(experts) and rt.expert_budget == 0 and rt.pack_budget == others + own
    model, rt = bound8(monkeypatch, config, 2 * others + own + each - 1)
    assert sum(e is not None for e in experts_of(model)) == len(experts) - 1


def test_a_model_that_fits_in_8_bits_alone_keeps_its_copies(monkeypatch):
    """What is free when a model is about to be bound has to hold its matrices as they will be: one that has no room in bfloat16 may have room in 8 bits, and the
    head its copy."""
    layer = tiny_configs.ALL["layer_8b"]
    model = model_of(dict(layer, vocab_size=512))
    native, own = step._own_bytes(model, torch.bfloat16, 64), step._own_bytes(model, torch.bfloat16, 64, True)
    assert own < 0.6 * native
    free = (native + own) // 2
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda: (free, 0))
    monkeypatch.setattr(torch.cuda, "memory_reserved", lambda: 0)
    monkeypatch.setattr(torch.cuda, "memory_allocated", lambda: 0)
    room = lambda *eight: step.packed_weight_budget(model, torch.bfloat16, 64, torch.device("cpu"), *eight)  # noqa: E731
    assert room() == 0 and room(True) == free - own
    rt = base.Runtime(torch.device("cpu"), torch.bfloat16, eight_bit=True)
    step._packing(rt, model, 64, None)
    assert rt.pack_budget == free - own >= model.packable_bytes(True) == model.head.packable_bytes()


@pytest.mark.parametrize("call", [lambda l, a: l.product(a), lambda l, a: l.product(a, rows_out=64), lambda l, a: l.product(a, f32_ok=True), lambda l, a: l.forward(a)])
@pytest.mark.parametrize("rows", [lambda: torch.zeros(3, 128, dtype=torch.bfloat16), lambda: torch.zeros(3, 128), lambda: K.BlockRows(3, 128, torch.empty(0))])
def test_gate_and_up_in_8_bits_give_their_product_only(call, rows):
    """A stacked gate and up matrix in 8 bits lies in the order of silu(gate) * up: the rows [gate | up] that product() and forward() are for cannot be had of it."""
    linear = importlib.import_module("daisi-llogos_amd.parts.linear").Linear(["g", "u"], 128, [64, 64], gated=True, eight_bit=True)
    linear.rt = base.Runtime(torch.device("cpu"), torch.bfloat16, eight_bit=True)
    linear.block = K.BlockWeight(torch.zeros(128 * 64, dtype=torch.bfloat16), torch.ones(2, 1, 4, dtype=torch.uint8), 128, 128, 64)
    with pytest.raises(K.KernelError, match="gated_product"):
        call(linear, rows())


def test_whether_matrices_come_from_memory(monkeypatch):
    """A model that is larger than the last-level cache says so to its matrices in 8 bits, whatever their own size is; a smaller one does not."""
    config = peponex_configs.PEP_C
    for small, large in ((1 << 10, False), (1 << 30, True)):
        model, _ = bound8(monkeypatch, config, 1 << 40)
        held = sum(p.weight_bytes() for p in model.layers + model.stream_parts) + model.head.weight_bytes()
        assert (1 << 10) < held < (1 << 30)
        monkeypatch.setattr(K, "LAST_LEVEL_CACHE", small)
        model, _ = bound8(monkeypatch, config, 1 << 40)
        blocks = [l.block for layer in model.layers for l in linears(layer) if l.block is not None]
        assert blocks and all(b.once is not large for b in blocks)
    w = K.BlockWeight(torch.zeros(2 * 64 * 64, dtype=torch.bfloat16), torch.ones(2, 1, 4, dtype=torch.uint8), 128, 128, once=True)
    assert w.rows(64).once and w.rows(128).once


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 20401, 40401, 40403, 20805, 10401, 1])
@pytest.mark.parametrize("M", [20, 61, 130, 300])
@pytest.mark.parametrize("gate_rows", [0, 160])
def test_a_matrix_from_memory_gives_the_same(form, M, gate_rows):
    g = torch.Generator(device="cuda").manual_seed(form + M)
    a, w = torch.randn(M, 1600, generator=g, device="cuda"), torch.randn(320, 1600, generator=g, device="cuda")
    rows, matrix = K.quantize_rows(a), K.quantize_weight(w)
    one, other = (K.block_weight(*matrix, gate_rows=gate_rows, once=o) for o in (False, True))
    assert other.once and not one.once
    assert torch.equal(K.gemm_blocks(rows, one, form=form), K.gemm_blocks(rows, other, form=form))
    assert torch.equal(K.gemm_blocks(rows, one, form=form, sums_ok=True), K.gemm_blocks(rows, other, form=form, sums_ok=True))
