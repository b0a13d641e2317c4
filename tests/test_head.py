"""Refusals of the retrieval head's operators, the C entry points' checks, and
the module's buffers: no GPU needed."""

import pytest
import torch

import silvertorch_amd.ops._load_ops  # noqa: F401
from silvertorch_amd import capi

st = torch.ops.st


def _raises(message, call):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_target_logprobs_refusals():
    z, t = torch.zeros((2, 70)), torch.zeros(2, dtype=torch.long)
    _raises("2-D", lambda: st.target_logprobs(z[0], t))
    _raises("float32, float16 or bfloat16", lambda: st.target_logprobs(z.double(), t))
    _raises("1-D int64", lambda: st.target_logprobs(z, t.int()))
    _raises("1-D int64", lambda: st.target_logprobs(z, t.view(2, 1)))
    _raises("3 entries", lambda: st.target_logprobs(z, torch.zeros(3, dtype=torch.long)))
    for k in (-1, 129):
        _raises("topk", lambda: st.target_logprobs(z, t, k))
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-9):
        _raises("temperature", lambda: st.target_logprobs(z, t, 0, None, temperature))
    _raises("packed search output", lambda: st.target_logprobs(z, t, 0, torch.zeros((2, 2), dtype=torch.int32)))
    _raises("packed search output", lambda: st.target_logprobs(z, t, 0, torch.zeros(2, dtype=torch.long)))
    _raises("3 rows", lambda: st.target_logprobs(z, t, 0, torch.zeros((3, 2), dtype=torch.long)))
    _raises("64 documents", lambda: st.target_logprobs(z, t, 0, torch.zeros((2, 1), dtype=torch.long)))
    _raises("topk", lambda: st.target_logprobs(z.clone().requires_grad_(), t, 129))


def test_cluster_route_refusals():
    z = torch.zeros((4, 9))
    _raises("2-D", lambda: st.cluster_route(z[0], 2))
    _raises("float32, float16 or bfloat16", lambda: st.cluster_route(z.long(), 2))
    for k in (0, 65):
        _raises("probes", lambda: st.cluster_route(z, k))
    _raises("clusters", lambda: st.cluster_route(torch.zeros((4, 0)), 1))
    _raises("clusters", lambda: st.cluster_route(torch.zeros((1, 32_769)), 1))
    _raises("bool", lambda: st.cluster_route(z, 2, torch.ones(4)))
    _raises("bool", lambda: st.cluster_route(z, 2, torch.ones(3, dtype=torch.bool)))


def test_int4_refusals():
    p, s, x = torch.zeros((5, 32), dtype=torch.uint8), torch.ones((5, 2)), torch.ones((3, 40))
    for g in (0, 16, 33, -32):
        _raises("group_size", lambda: st.int4_matvec(p, s, x, g))
        _raises("group_size", lambda: st.int4_quantize(x, g))
    _raises("uint8", lambda: st.int4_matvec(p.int(), s, x, 32))
    _raises("bytes a row", lambda: st.int4_matvec(p, s, torch.ones((3, 70)), 32))
    _raises("scales must be", lambda: st.int4_matvec(p, s[:, :1], x, 32))
    _raises("zeros", lambda: st.int4_matvec(p, s, x, 32, torch.zeros((5, 2))))
    _raises("zeros", lambda: st.int4_matvec(p, s, x, 32, torch.zeros((5, 1), dtype=torch.uint8)))
    _raises("float32, float16 or bfloat16", lambda: st.int4_matvec(p, s, x, 32, None, torch.float64))
    _raises("float32, float16 or bfloat16", lambda: st.int4_matvec(p, s, x.long(), 32))
    _raises("float32, float16 or bfloat16", lambda: st.int4_matvec(p, s.double(), x, 32))
    _raises("vector", lambda: st.int4_matvec(p, s, x.view(1, 3, 40), 32))
    _raises("at least one column", lambda: st.int4_matvec(p[:, :0], s[:, :0], x[:, :0], 32))
    _raises("2-D", lambda: st.int4_quantize(x[0], 32))


def test_c_entry_points_refuse():
    """Status codes and messages, before any device work."""
    L = capi.lib()

    def refused(message, rc):
        assert rc != 0
        assert message in L.st_last_error().decode()

    n = None
    refused("group_size", L.st_int4_matvec(n, n, 0, n, n, 0, 1, 1, 64, 31, n, 0, n))
    refused("scales", L.st_int4_matvec(n, n, 5, n, n, 0, 1, 1, 64, 32, n, 0, n))
    refused("null device pointer", L.st_int4_matvec(n, n, 0, n, n, 0, 1, 1, 64, 32, n, 0, n))
    refused("16-byte aligned", L.st_int4_matvec(8, 16, 0, n, 16, 0, 1, 1, 64, 32, 16, 0, n))
    refused("between 0 and 65536", L.st_int4_matvec(16, 16, 0, n, 16, 0, 65_537, 1, 64, 32, 16, 0, n))
    refused("at least one column", L.st_int4_quantize(n, 0, 1, 0, 32, 1, n, n, n, n))
    refused("topk", L.st_target_logprobs(n, 0, 1, 5, 5, n, n, 0, 0, 200, 1.0, *[n] * 8))
    refused("temperature", L.st_target_logprobs(n, 0, 1, 5, 5, n, n, 0, 0, 2, 0.0, *[n] * 8))
    refused("null device pointer", L.st_target_logprobs(n, 0, 1, 5, 5, n, n, 0, 0, 2, 1.0, *[n] * 8))
    refused("fewer than", L.st_target_logprobs(16, 0, 1, 65, 65, 16, 16, 1, 1, 2, 1.0, *[n] * 8))
    refused("2^31", L.st_target_logprobs(16, 0, 1, 1 << 31, 1 << 31, 16, n, 0, 0, 2, 1.0, *[n] * 8))
    refused("null device pointer", L.st_target_logprobs_backward(16, 0, 1, 5, 5, 16, n, 0, 0, 2, 1.0, *[n] * 9))
    refused("probes", L.st_cluster_route(n, 0, 1, 5, 5, 0, *[n] * 10))
    refused("clusters", L.st_cluster_route(n, 0, 1, 40_000, 5, 1, *[n] * 10))
    refused("below 2^31", L.st_cluster_route(n, 0, 1 << 31, 5, 5, 1, *[n] * 10))
    refused("null device pointer", L.st_cluster_route(n, 0, 1, 5, 5, 1, *[n] * 10))
    refused("null device pointer", L.st_cluster_route_backward(n, 0, 1, 5, 5, 1, *[n] * 9))
    assert L.st_target_logprobs(n, 0, 0, 5, 5, n, n, 0, 0, 2, 1.0, *[n] * 8) == 0


def test_module_state():
    """The table's buffers take a saved table's sizes and types."""
    from silvertorch_amd.modules import RetrievalHeadModule

    a, b = RetrievalHeadModule(64, 5, 0.5), RetrievalHeadModule(64, 5, 0.5)
    a.set_table(torch.ones((7, 48), dtype=torch.uint8), torch.ones((7, 2), dtype=torch.bfloat16),
                torch.full((7, 2), 8, dtype=torch.uint8))
    b.load_state_dict(a.state_dict())
    assert b.packed.shape == (7, 48) and b.scales.dtype == torch.bfloat16 and torch.equal(b.zeros, a.zeros)
