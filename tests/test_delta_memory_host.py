"""DeltaMemory's parts that need no GPU."""
import math

import pytest
import torch

from flyguy_b200 import delta


@pytest.mark.parametrize("dim", [9, 16, 32, 40, 64, 81, 96, 128])
def test_keys_are_no_longer_than_one_whatever_is_learned(dim):
    """A normed key x has |x|^2 <= dim, so that |x w|^2 <= dim max(w)^2. At first, and below, the weight is taken as it is, its
    gradient too; beyond, as much of it as keeps the bound, and its gradient is that of differences."""
    m = delta.DeltaMemory(8, 4, heads=2, key_heads=1, dim=dim)
    g = torch.arange(1.0, dim + 1)
    assert torch.equal(m._key_weight(), m.k_weight)
    assert torch.equal(torch.autograd.grad(m._key_weight(), m.k_weight, g)[0], g)
    with torch.no_grad():
        m.k_weight.copy_(torch.linspace(-0.5, 0.9, dim) * dim ** -0.5)
    assert torch.equal(m._key_weight(), m.k_weight)
    for by in (4.0, 1e6):
        with torch.no_grad():
            m.k_weight.copy_(torch.linspace(-by, by / 2, dim))
        w = m._key_weight()
        assert dim * w.abs().max().item() ** 2 <= 1 + 1e-6
        assert torch.allclose(w / w.abs().max(), m.k_weight / m.k_weight.abs().max())
    with torch.no_grad():
        m.k_weight.fill_(math.nan)
    assert m._key_weight().isnan().all()
    m = m.double()
    with torch.no_grad():
        m.k_weight.copy_(torch.linspace(-1.0, 2.0, dim))
    got, = torch.autograd.grad((m._key_weight() * g).sum(), m.k_weight)
    for i in (0, dim - 1):
        with torch.no_grad():
            ends = []
            for step in (1e-6, -2e-6):
                m.k_weight[i] += step
                ends.append((m._key_weight() * g).sum())
        assert abs((ends[0] - ends[1]) / 2e-6 - got[i]) <= 1e-6 * g.sum()
        with torch.no_grad():
            m.k_weight[i] += 1e-6


def test_a_saved_memory_goes_on_counting_its_calls():
    """Loaded, by itself and inside another module, it drops where it had come to; a dictionary of before the count loads, too."""
    m, other = (delta.DeltaMemory(8, 4, heads=2, key_heads=1, dim=16, dropout=0.1) for _ in range(2))
    m.calls = 41
    saved = m.state_dict()
    other.load_state_dict(saved)
    assert other.calls == 41
    m.calls = 5
    inside = torch.nn.Sequential(torch.nn.Linear(8, 8), other)
    inside.load_state_dict(torch.nn.Sequential(torch.nn.Linear(8, 8), m).state_dict())
    assert other.calls == 5
    del saved["calls"]
    other.load_state_dict(saved)
    assert other.calls == 5
    with pytest.raises(RuntimeError, match="Unexpected"):
        other.load_state_dict(saved | {"cells": torch.tensor(1)})


def test_a_memory_pickled_whole_has_all_that_it_needs():
    """Its own attributes are those that a memory pickled before had."""
    own = set(vars(delta.DeltaMemory(8, 4, heads=2, key_heads=1, dim=16))) - set(vars(torch.nn.Module()))
    assert own == {"heads", "key_heads", "dim", "dtype", "dropout", "seed", "calls"}
