"""How the operators beside the projections are reached: every package of popxl_addons.ops is a module with its public names,
also where one of them is a function of the module's own name, which the module then can be called as."""
import inspect
import os
import subprocess
import sys
import types

import pytest
import torch

import popxl_addons.ops
from popxl_addons.ops import kv_cache_gq, low_rank_adapters, rotary_pos_embed

PACKAGES = (kv_cache_gq, low_rank_adapters, rotary_pos_embed)


@pytest.mark.parametrize("package", PACKAGES, ids=lambda p: p.__name__)
def test_packages_are_modules_with_their_names(package):
    assert isinstance(package, types.ModuleType) and sys.modules[package.__name__] is package
    inner = sys.modules[package.__name__ + "." + package.__name__.rpartition(".")[2]]
    for name in inner.__all__:
        assert getattr(package, name) is getattr(inner, name), name


@pytest.mark.parametrize("package", PACKAGES, ids=lambda p: p.__name__)
def test_public_names_are_in_the_namespace_of_the_operators(package):
    own = package.__name__.rpartition(".")[2]
    for name in sys.modules[f"{package.__name__}.{own}"].__all__:
        if name not in (own, "BLOCK_SIZE"):
            assert getattr(popxl_addons.ops, name) is getattr(package, name), name


@pytest.mark.parametrize("package", PACKAGES[1:], ids=lambda p: p.__name__)
def test_module_is_called_as_its_function(package):
    function = getattr(package, package.__name__.rpartition(".")[2])
    assert isinstance(function, types.FunctionType) and callable(package)
    assert inspect.signature(package) == inspect.signature(function)
    assert function.__doc__ and package.__wrapped__ is function


def test_calls_through_either_name_are_the_same():
    rotary, t = rotary_pos_embed.RotaryPosEmbed(32, device="cpu"), torch.zeros((3, 2, 64), dtype=torch.float16)
    for call in (rotary_pos_embed, rotary_pos_embed.rotary_pos_embed, popxl_addons.ops.rotary_pos_embed):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(t, torch.zeros(3, dtype=torch.int32), rotary)
        with pytest.raises(TypeError):
            call(t)


@pytest.mark.parametrize("line", ["from popxl_addons.ops import rotary_pos_embed", "import popxl_addons.ops.rotary_pos_embed as rotary_pos_embed",
                                  "from popxl_addons.layers.linear_gq import LinearGQ; from popxl_addons.ops import rotary_pos_embed",
                                  "from popxl_addons.ops.low_rank_adapters import low_rank_adapters; from popxl_addons.ops import rotary_pos_embed"])
def test_whatever_is_imported_first(line):
    check = "assert callable(rotary_pos_embed) and rotary_pos_embed.RotaryPosEmbed and rotary_pos_embed.rotary_pos_embed"
    path = os.path.dirname(os.path.dirname(popxl_addons.__file__))
    subprocess.run([sys.executable, "-c", f"{line}; {check}"], check=True, env={**os.environ, "PYTHONPATH": path})
