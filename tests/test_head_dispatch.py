"""The retrieval head's differentiable operators go through the dispatcher, with
and without gradients (tests/test_tower_dispatch.py says how these tests run
without a GPU)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

import silvertorch_amd.ops._load_ops  # noqa: F401

st = torch.ops.st


class Answers(TorchDispatchMode):
    """Names of st operators, answered with tensors of ones of the right shapes."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace != "st":
            return func(*args, **(kwargs or {}))
        name = func._schema.name.removeprefix("st::")
        self.seen.append(name)
        self.args = args
        n, ones = len(args[0]), torch.ones
        if name.endswith("_backward"):
            return torch.full_like(args[0], 2.0)
        if name.startswith("target_logprobs"):
            topk = args[2] if len(args) > 2 else 0
            out = [ones(n), ones(n), ones(n), ones((n, topk), dtype=torch.long), ones((n, topk))]
            return (*out, ones((n, 2))) if name.endswith("_with_stats") else tuple(out)
        assert name.startswith("cluster_route")
        columns, probes = args[0].shape[1], args[1]
        out = [ones((n, probes), dtype=torch.long), ones((n, probes)), ones(n), ones(columns, dtype=torch.long), ones(())]
        return (*out, ones((n, 2)), ones(columns)) if name.endswith("_with_stats") else tuple(out)


@pytest.mark.parametrize("grad", [False, True])
def test_a_mode_sees_target_logprobs(grad):
    z = torch.ones((3, 70), requires_grad=grad)
    targets, mask = torch.zeros(3, dtype=torch.long), torch.ones((3, 32), dtype=torch.long)
    for m in (None, mask):
        with Answers() as mode:
            out = st.target_logprobs(z, targets, 4, m, 0.5)
            if grad:
                g, = torch.autograd.grad(out[0].sum() + out[4].sum(), z)
                assert (g == 2).all()
        assert mode.seen == (["target_logprobs_with_stats", "target_logprobs_backward"] if grad else ["target_logprobs"])
        if grad:
            assert [a is not None for a in mode.args[8:]] == [True, False, False, True] and (mode.args[3] is None) == (m is None)


@pytest.mark.parametrize("grad", [False, True])
def test_a_mode_sees_cluster_route(grad):
    z = torch.ones((3, 70), requires_grad=grad)
    with Answers() as mode:
        out = st.cluster_route(z, 4, torch.tensor([True, False, True]))
        if grad:
            g, = torch.autograd.grad(out[1].sum() + out[4], z)
            assert (g == 2).all()
    assert mode.seen == (["cluster_route_with_stats", "cluster_route_backward"] if grad else ["cluster_route"])
    if grad:
        assert [a is not None for a in mode.args[5:]] == [True, False, True]


def test_fake_scores_do_not_reach_a_kernel():
    for grad in (False, True):
        mode = FakeTensorMode()
        z, targets = torch.ones((3, 70), requires_grad=grad), torch.zeros(3, dtype=torch.long)
        with mode, pytest.raises(Exception, match=r"st\.|st::"):
            st.target_logprobs(mode.from_tensor(z), mode.from_tensor(targets), 4)
        with mode, pytest.raises(Exception, match=r"st\.|st::"):
            st.cluster_route(mode.from_tensor(z), 4)


def test_target_logprobs_backward_refusals():
    z, t = torch.zeros((3, 70)), torch.zeros(3, dtype=torch.long)
    one, ids, two = torch.zeros(3), torch.zeros((3, 4), dtype=torch.long), torch.zeros((3, 2))

    def refused(message, topk=4, entropy=one, top_ids=ids, stats=two, grads=(None, None, None, None), temperature=1.0):
        with pytest.raises(RuntimeError, match=message):
            st.target_logprobs_backward(z, t, topk, None, temperature, entropy, top_ids, stats, *grads)

    refused("entropy must be", entropy=one[:2])
    refused("top_ids must be", topk=5)
    refused("top_ids must be", top_ids=ids.int())
    refused("stats must be", stats=two.double())
    refused("gradients must be", grads=(two, None, None, None))
    refused("gradients must be", grads=(None, None, None, two))
    refused("gradients must be", grads=(None, None, one[:2], None))
    refused("temperature", temperature=0.0)


def test_cluster_route_backward_refusals():
    z = torch.zeros((3, 70))
    ids, four, two, slopes = torch.zeros((3, 4), dtype=torch.long), torch.zeros((3, 4)), torch.zeros((3, 2)), torch.zeros(70)

    def refused(message, logits=z, ids=ids, weights=four, stats=two, slopes=slopes, grads=(None, None, None)):
        with pytest.raises(RuntimeError, match=message):
            st.cluster_route_backward(logits, ids, weights, stats, slopes, *grads)

    refused("logits must be a 2-D", logits=z[0])
    refused("probes must be", ids=torch.zeros((3, 65), dtype=torch.long))
    refused("cluster_ids must be", ids=ids.int())
    refused("cluster_ids must be", ids=ids[:2])
    refused("weights must be", weights=four[:, :3])
    refused("stats must be", stats=four)
    refused("slopes must be", slopes=slopes[:69])
    refused("gradients must be", grads=(two, None, None))
    refused("gradients must be", grads=(None, two, None))
    refused("gradients must be", grads=(None, None, two))
