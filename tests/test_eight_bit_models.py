"""Models under weights='fp8' without a GPU: which are refused, and what memory their matrices are counted on to take."""
import importlib

import pytest

import nipulorn_configs
import peponex_configs
import tiny_configs
import zasidra_configs
import zogurax_configs

L = importlib.import_module("daisi-llogos_amd")
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
