"""Activation checkpointing of the query tower on the GPU: a checkpointed pass
has the embeddings and the gradients of the same pass kept whole.

Tolerance: the same products and kernels on the same inputs run twice; a
library's product may choose another order of its sums, as in
test_gpu_tower_modules.py, 2^-10 of a result's 2-norm."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests import gpu_helpers as H
from tests.test_gpu_tower_modules import _close, _tower

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_checkpointed_training_pass(use_reentrant):
    H.note(f"[tower] checkpoint {use_reentrant}")
    tower, other = _tower(), _tower()
    x = torch.randn((50, 24), generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    y = x.detach().clone().requires_grad_()
    for _ in range(2):
        want = tower(x)
        out = checkpoint(other, y, other.next_state(), use_reentrant=use_reentrant)
        _close(out, want.cpu(), 2.0 ** -10)
        want.square().sum().backward()
        out.square().sum().backward()
    assert torch.equal(tower.rng, other.rng)
    for a, b in zip([y, *other.parameters()], [x, *tower.parameters()]):
        _close(a.grad, b.grad.cpu(), 2.0 ** -10)


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_checkpointed_training_pass_without_a_state_is_refused(use_reentrant):
    H.note(f"[tower] checkpoint without a state {use_reentrant}")
    tower = _tower()
    x = torch.randn((50, 24), generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    out = checkpoint(tower, x, use_reentrant=use_reentrant)
    with pytest.raises(RuntimeError, match="give it a state"):
        out.square().sum().backward()
