"""adapter_linear keeps no graph: operands that would need one are refused, before anything looks at where they live."""
import pytest
import torch

from flatland_marl_amd import FlmError
from flatland_marl_amd.adapters import RowGroups, adapter_linear

NAMES = ("x", "weight", "bias", "a", "b")


def _operands(**requires):
    f = torch.zeros
    t = dict(x=f(4, 8), weight=f(6, 8), bias=f(6), a=f(2, 3, 8), b=f(2, 6, 3))
    return {name: v.requires_grad_(requires.get(name, False)) for name, v in t.items()}


def _call(t):
    return adapter_linear(t["x"], t["weight"], t["bias"], t["a"], t["b"], RowGroups(torch.zeros(20, dtype=torch.int32), 4, 2))


@pytest.mark.parametrize("name", NAMES)
def test_operands_that_require_a_gradient(name):
    t = _operands(**{name: True})
    with pytest.raises(ValueError, match="no_grad"):
        _call(t)
    # the same call without a graph to record gets as far as the missing GPU
    with torch.no_grad(), pytest.raises(FlmError):
        _call(t)
    with pytest.raises(FlmError):
        _call({k: v.detach() for k, v in t.items()})


def test_operands_without_gradients_and_without_bias():
    t = _operands()
    t["bias"] = None
    with pytest.raises(FlmError):
        _call(t)
