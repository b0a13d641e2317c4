"""The retrieval head's operators and forward-mode derivatives: no GPU needed, an input with a tangent is refused
before any device work."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import silvertorch_amd.ops._load_ops  # noqa: F401

st = torch.ops.st


def _calls():
    z, x = torch.zeros((2, 70)), torch.ones((3, 40))
    packed, scales = torch.zeros((5, 32), dtype=torch.uint8), torch.ones((5, 2))
    return {
        "target_logprobs": (z, lambda t: st.target_logprobs(t, torch.zeros(2, dtype=torch.long))),
        "cluster_route": (z, lambda t: st.cluster_route(t, 2)),
        "int4_matvec": (x, lambda t: st.int4_matvec(packed, scales, t, 32)),
        "int4_matvec with scales": (scales, lambda t: st.int4_matvec(packed, t, x, 32)),
        "int4_quantize": (x, lambda t: st.int4_quantize(t, 32)),
    }


@pytest.mark.parametrize("name", list(_calls()))
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_tangents_are_refused(name, requires_grad, grad_mode):
    value, call = _calls()[name]
    message = f"{name.split()[0]} has no forward-mode derivative"
    with fwAD.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fwAD.make_dual(value.clone().requires_grad_(requires_grad), torch.ones_like(value))
        with pytest.raises(RuntimeError, match=message):
            call(dual)
