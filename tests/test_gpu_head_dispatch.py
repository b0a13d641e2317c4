"""The operators that the retrieval head's gradients call, by themselves on the
GPU: the gradients that autograd gives, and ids that are no cluster's."""

import pytest
import torch

from tests import gpu_helpers as H

pytestmark = pytest.mark.gpu
st = torch.ops.st


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _scores(rows, columns, seed):
    return torch.randn((rows, columns), generator=torch.Generator().manual_seed(seed)).cuda().requires_grad_()


@pytest.mark.parametrize("columns", [70, 700, 20_000])
def test_target_logprobs_backward_is_autograds(columns):
    H.note(f"[head] target_logprobs_backward {columns}")
    z = _scores(5, columns, 1)
    targets = torch.tensor([0, 3, columns - 1, -1, 7]).cuda()
    gl, gt = _scores(1, 5, 2)[0].detach(), _scores(5, 4, 3).detach()
    out = st.target_logprobs(z, targets, 4, None, 0.5)
    want, = torch.autograd.grad([out[0], out[4]], z, [gl, gt])
    flat = z.detach()
    kept = st.target_logprobs_with_stats(flat, targets, 4, None, 0.5)
    assert all(torch.equal(a, b) for a, b in zip(out, kept))
    got = st.target_logprobs_backward(flat, targets, 4, None, 0.5, kept[1], kept[3], kept[5], gl, None, None, gt)
    assert torch.equal(got, want)


@pytest.mark.parametrize("columns", [70, 300, 700, 5000, 20_000])
def test_cluster_route_backward_is_autograds(columns):
    H.note(f"[head] cluster_route_backward {columns}")
    z = _scores(37, columns, 1)
    gw, gs = _scores(37, 4, 2).detach(), _scores(1, 37, 3)[0].detach()
    out = st.cluster_route(z, 4)
    want, = torch.autograd.grad([out[1], out[2]], z, [gw, gs])
    kept = st.cluster_route_with_stats(z.detach(), 4, None)
    back = lambda ids: st.cluster_route_backward(z.detach(), ids, kept[1], kept[5], kept[6], gw, gs, None)  # noqa: E731
    assert torch.equal(back(kept[0]), want)
    # an id that is no cluster's is none
    none = kept[0].clone()
    none[::2, 1] = -1
    for other in (columns, 1 << 40, -(1 << 32), -7):
        ids = kept[0].clone()
        ids[::2, 1] = other
        assert torch.equal(back(ids), back(none))
