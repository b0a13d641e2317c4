"""Activation checkpointing of the query tower without a GPU: plain operators
stand in for the kernels, so only which state a pass takes is tested."""

import types

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from silvertorch_amd.modules import QueryTowerModule
from tests import tower_oracle as O


@pytest.fixture
def plain(monkeypatch):
    def dropout(x, p, state):
        return torch.where(O.keeps(x.shape, p, state.tolist()), x * O.times(p), 0.0)

    def dropout_add_layer_norm(x, residual, weight, bias, p, state, eps):
        h = residual + (dropout(x, p, state) if p else x)
        return O.layer_norm(h, weight, bias, eps), h

    st = types.SimpleNamespace(dropout=dropout, layer_norm=O.layer_norm, dropout_add_layer_norm=dropout_add_layer_norm)
    monkeypatch.setattr(torch.ops, "st", st, raising=False)


def _tower():
    torch.manual_seed(0)
    return QueryTowerModule(6, 8, 16, layers=2, expand=2, dropout=0.4, seed=9).double()


def _gradients(tower, out):
    return torch.autograd.grad(out.square().sum(), list(tower.parameters()))


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_checkpointed_pass_with_its_state(plain, use_reentrant):
    """Two passes ahead of their backward passes: outputs, gradients and the state afterwards are those of plain passes."""
    x = torch.randn((2, 5, 6), dtype=torch.float64, requires_grad=True)
    tower, other = _tower(), _tower()
    want = [tower(x[i]) for i in range(2)]
    params = list(other.parameters())
    got = [checkpoint(other, x[i], other.next_state(), use_reentrant=use_reentrant) for i in range(2)]
    assert torch.equal(tower.rng, other.rng) and other.rng.tolist() == [9, 6]
    for a, b in zip(want, got):
        assert torch.equal(a, b)
        b.square().sum().backward()
        for p, g in zip(params, _gradients(tower, a)):
            assert torch.equal(p.grad, g)
            p.grad = None
    assert other.rng.tolist() == [9, 6]


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_checkpointed_pass_without_a_state_is_refused(plain, use_reentrant):
    tower = _tower()
    x = torch.randn((5, 6), dtype=torch.float64, requires_grad=True)
    out = checkpoint(tower, x, use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="give it a state"):
        out.square().sum().backward()
    assert tower.rng.tolist() == [9, 3]


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_checkpointed_pass_without_dropout(plain, use_reentrant):
    tower = _tower().eval()
    x = torch.randn((5, 6), dtype=torch.float64, requires_grad=True)
    want = _gradients(tower, tower(x))
    checkpoint(tower, x, use_reentrant=use_reentrant).square().sum().backward()
    assert all(torch.equal(p.grad, g) for p, g in zip(tower.parameters(), want))
    assert tower.rng.tolist() == [9, 0]


def test_states_of_other_shapes_are_refused(plain):
    tower, x = _tower(), torch.zeros((5, 6), dtype=torch.float64)
    for state in (tower.rng[:1], tower.places, tower.rng[0]):
        with pytest.raises(RuntimeError, match="seed and offset"):
            tower(x, state)
