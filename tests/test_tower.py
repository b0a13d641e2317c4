"""The query tower's operators without a GPU: their refusals, the C entry
points' checks, forward-mode derivatives, the oracle's random numbers."""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import silvertorch_amd.ops._load_ops  # noqa: F401
from silvertorch_amd import capi
from tests import tower_oracle as O

st = torch.ops.st


def _raises(message, call):
    with pytest.raises(RuntimeError, match=message):
        call()


@pytest.mark.parametrize("counter,key,want", [
    ([0, 0, 0, 0], [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_generator_gives_the_published_words(counter, key, want):
    assert [int(w) for w in O.philox(counter, key)] == want


def test_kept_share():
    """2^20 draws: the share that stays is within 5 standard deviations of 1 - p in units of 2^-16."""
    n = 1 << 20
    for p in (0.1, 0.5, 0.9):
        q = 1 - O.units(p) / 65536
        share = O.keeps((n,), p, (3, 5)).double().mean().item()
        assert abs(share - q) < 5 * np.sqrt(q * (1 - q) / n)


def test_layer_norm_refusals():
    x, w = torch.zeros((3, 10)), torch.ones(10)
    _raises("float32, float16 or bfloat16", lambda: st.layer_norm(x.double()))
    _raises("float32, float16 or bfloat16", lambda: st.layer_norm(x, w.double()))
    _raises("at least one dimension", lambda: st.layer_norm(x[0, 0]))
    _raises("between 1 and 32768", lambda: st.layer_norm(torch.zeros((2, 0))))
    _raises("between 1 and 32768", lambda: st.layer_norm(torch.zeros((1, 32_769))))
    _raises("one entry", lambda: st.layer_norm(x, w[:9]))
    _raises("one entry", lambda: st.layer_norm(x, w, w.view(10, 1)))
    _raises("of one type", lambda: st.layer_norm(x, w, w.half()))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        _raises("eps", lambda: st.layer_norm(x, w, w, eps))
        _raises("eps", lambda: st.layer_norm_int8(x, w, w, eps))
    _raises("one entry", lambda: st.layer_norm_int8(x, w[:9]))
    _raises("between 1 and 32768", lambda: st.layer_norm_int8(torch.zeros((1, 32_769))))


def test_dropout_refusals():
    x, s = torch.zeros((3, 10)), torch.zeros(2, dtype=torch.long)
    for p in (-0.1, 1.5, float("nan")):
        _raises(r"p must be in \[0, 1\]", lambda: st.dropout(x, p, s))
        _raises(r"p must be in \[0, 1\]", lambda: st.dropout_add_layer_norm(x, x, None, None, p, s))
    _raises("seed and offset", lambda: st.dropout(x, 0.5, s.int()))
    _raises("seed and offset", lambda: st.dropout(x, 0.5, s[:1]))
    _raises("seed and offset", lambda: st.dropout_add_layer_norm(x, x, None, None, 0.5, s.view(1, 2)))
    _raises("float32, float16 or bfloat16", lambda: st.dropout(x.long(), 0.5, s))
    _raises("needs a state", lambda: st.dropout_add_layer_norm(x, x, None, None, 0.5))
    _raises("x's shape", lambda: st.dropout_add_layer_norm(x, x[:1]))
    _raises("x's type or float32", lambda: st.dropout_add_layer_norm(x, x.half()))
    _raises("x's type or float32", lambda: st.dropout_add_layer_norm(x.bfloat16(), x.half()))


def test_int8_refusals():
    t, s = torch.zeros((5, 32), dtype=torch.int8), torch.ones(5)
    x, xs = torch.zeros((3, 20)), torch.ones(3)
    codes = torch.zeros((3, 32), dtype=torch.int8)
    _raises("at least one column", lambda: st.int8_quantize(torch.zeros((3, 0))))
    _raises("float32, float16 or bfloat16", lambda: st.int8_quantize(x.double()))
    _raises("2-D int8", lambda: st.int8_matmul(t.int(), s, x))
    _raises("2-D int8", lambda: st.int8_matmul(t[0], s, x))
    _raises("blocks of 16", lambda: st.int8_matmul(t[:, :20], s, x))
    _raises("vectors of 33 take 48", lambda: st.int8_matmul(t, s, torch.zeros((3, 33))))
    _raises("vectors of 16 take 16", lambda: st.int8_matmul(t, s, torch.zeros((3, 16))))
    _raises("rows of 16 codes", lambda: st.int8_matmul(t, s, codes[:, :16], xs))
    _raises("comes with x_scales", lambda: st.int8_matmul(t, s, codes))
    _raises("x_scales go with", lambda: st.int8_matmul(t, s, x, xs))
    _raises("x_scales must be", lambda: st.int8_matmul(t, s, codes, xs[:2]))
    _raises("x_scales must be", lambda: st.int8_matmul(t, s, codes, xs.double()))
    _raises("scales must be", lambda: st.int8_matmul(t, s[:4], x))
    _raises("scales must be", lambda: st.int8_matmul(t, s.half(), x))
    _raises("bias must be", lambda: st.int8_matmul(t, s, x, None, s.half()))
    _raises("bias must be", lambda: st.int8_matmul(t, s, x, None, s[:3]))
    _raises("float32, float16 or bfloat16", lambda: st.int8_matmul(t, s, x.long()))
    _raises("out_dtype must be", lambda: st.int8_matmul(t, s, x, None, None, torch.float64))


def test_c_entry_points_refuse():
    """Status codes and messages, before any device work."""
    L = capi.lib()
    n = None

    def refused(message, rc):
        assert rc != 0
        assert message in L.st_last_error().decode()

    refused("float32, float16", L.st_dropout(n, 3, 1, 0.5, n, n, n, n))
    refused("p must be", L.st_dropout(n, 0, 1, 1.5, n, n, n, n))
    refused("negative", L.st_dropout(n, 0, -1, 0.5, n, n, n, n))
    refused("null device pointer", L.st_dropout(16, 0, 1, 0.5, n, 16, n, n))
    assert L.st_dropout(n, 0, 0, 0.5, n, n, n, n) == 0
    norm = lambda x=16, xt=0, rows=1, dim=8, res=n, rt=0, wt=0, eps=1e-5, p=0.0, state=n, y=16, total=n, used=n: (  # noqa: E731
        L.st_layer_norm(x, xt, rows, dim, dim, res, rt, dim, n, n, wt, eps, p, state, y, total, n, used, n))
    refused("x must be", norm(xt=4))
    refused("weight and bias must be", norm(wt=3))
    refused("columns must be", norm(dim=0))
    refused("columns must be", norm(dim=32_769))
    refused("negative", norm(rows=-1))
    refused("eps", norm(eps=0.0))
    refused("goes with a residual", norm(p=0.5))
    refused("needs a state", norm(res=16, p=0.5, total=16))
    refused("x's type or float32", norm(xt=2, res=16, rt=1, total=16))
    refused("null device pointer", norm(x=n))
    refused("null device pointer", norm(res=16))
    refused("null device pointer", norm(used=16))
    assert norm(rows=0, x=n) == 0
    back = lambda yt=0, ht=0, rows=1, dim=8, stats=16, p=0.0, ws=n, gx=16, gw=n: (  # noqa: E731
        L.st_layer_norm_backward(16, yt, n, 16, ht, rows, dim, dim, n, 0, stats, p, n, ws, gx, n, gw, n, n))
    refused("x's type or float32", back(yt=1, ht=2))
    refused("columns must be", back(dim=40_000))
    refused("null device pointer", back(stats=n))
    refused("null device pointer", back(gw=16))
    refused("needs a state", back(p=0.5))
    assert back(gx=n) == 0
    assert L.st_layer_norm_workspace_bytes(0, 8) == 0 and L.st_layer_norm_workspace_bytes(5, 40_000) == 0
    refused("16-byte aligned", L.st_layer_norm_int8(16, 0, 1, 8, 8, n, n, 0, 1e-5, 8, 16, n))
    refused("null device pointer", L.st_layer_norm_int8(16, 0, 1, 8, 8, n, n, 0, 1e-5, 16, n, n))
    assert [L.st_int8_columns(d) for d in (1, 16, 17)] == [16, 16, 32]
    refused("at least one column", L.st_int8_quantize(16, 0, 1, 0, 0, 16, 16, n))
    refused("blocks of 16", L.st_int8_quantize(16, 0, 1, 1 << 17, 1 << 17, 16, 16, n))
    mm = lambda t=16, cols=32, rows=4, x=16, xt=0, xs=n, tokens=2, dim=20, stride=20, y=16, yt=0: (  # noqa: E731
        L.st_int8_matmul(t, 16, rows, cols, x, xt, xs, tokens, dim, stride, n, y, yt, n, n))
    refused("blocks of 16", mm(cols=20))
    refused("blocks of 16", mm(cols=1 << 17, dim=1 << 17))
    refused("vectors of 33 take 48", mm(dim=33))
    refused("x must be", mm(xt=5))
    refused("the result must be", mm(yt=6))
    refused("16-byte aligned", mm(t=8))
    refused("null device pointer", mm(x=n))
    refused("side by side", mm(xt=6, xs=16))
    refused("come with scales", mm(xt=6, dim=32, stride=32))
    refused("negative", mm(tokens=-1))
    refused("negative", mm(rows=-1))
    assert mm(rows=0) == 0 and mm(tokens=0) == 0


def _calls():
    x, w, s = torch.ones((3, 40)), torch.ones(40), torch.zeros(2, dtype=torch.long)
    table, scales = torch.zeros((5, 48), dtype=torch.int8), torch.ones(5)
    codes, xs = torch.zeros((3, 48), dtype=torch.int8), torch.ones(3)
    return {
        "layer_norm": (x, lambda t: st.layer_norm(t, w)),
        "layer_norm with weight": (w, lambda t: st.layer_norm(x, t)),
        "dropout": (x, lambda t: st.dropout(t, 0.5, s)),
        "dropout_add_layer_norm": (x, lambda t: st.dropout_add_layer_norm(t, x)),
        "dropout_add_layer_norm with residual": (x, lambda t: st.dropout_add_layer_norm(x, t)),
        "int8_quantize": (x, lambda t: st.int8_quantize(t)),
        "layer_norm_int8": (x, lambda t: st.layer_norm_int8(t)),
        "int8_matmul": (x, lambda t: st.int8_matmul(table, scales, t)),
        "int8_matmul with scales": (scales, lambda t: st.int8_matmul(table, t, x)),
        "int8_matmul with x_scales": (xs, lambda t: st.int8_matmul(table, scales, codes, t)),
    }


@pytest.mark.parametrize("name", list(_calls()))
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(name, requires_grad):
    value, call = _calls()[name]
    with fwAD.dual_level():
        dual = fwAD.make_dual(value.clone().requires_grad_(requires_grad), torch.ones_like(value))
        with pytest.raises(RuntimeError, match=f"{name.split()[0]} has no forward-mode derivative"):
            call(dual)


def test_head_holds_an_eight_bit_table():
    """A table of `int8_quantize`, set or loaded, keeps its types; its scales stay float32."""
    from silvertorch_amd.modules import RetrievalHeadModule

    with pytest.raises(RuntimeError, match="bits must be 4 or 8"):
        RetrievalHeadModule(bits=3)
    a, b = RetrievalHeadModule(bits=8), RetrievalHeadModule()
    a.set_table(torch.ones((7, 48), dtype=torch.int8), torch.rand(7))
    b.load_state_dict(a.state_dict())
    assert b.packed.dtype == torch.int8 and b.packed.shape == (7, 48) and torch.equal(b.scales, a.scales)
    want = a.scales.clone()
    assert a.half().packed.dtype == torch.int8 and torch.equal(a.scales, want)
    four = RetrievalHeadModule()
    four.set_table(torch.ones((7, 16), dtype=torch.uint8), torch.rand((7, 1)), torch.full((7, 1), 8, dtype=torch.uint8))
    assert four.half().scales.dtype == torch.float16


def test_query_tower_state():
    """Parameters, dropout's state among the saved buffers, one state for each place that drops."""
    from silvertorch_amd.modules import QueryTowerModule

    a, b = QueryTowerModule(5, 8, 16, layers=3, seed=7), QueryTowerModule(5, 8, 16, layers=3)
    a.rng[1] += 12
    b.load_state_dict(a.state_dict())
    assert b.rng.tolist() == [7, 12] and "places" not in a.state_dict()
    assert (b.rng + b.places).tolist() == [[7, 12], [7, 13], [7, 14], [7, 15]]
    assert a.half().rng.dtype == torch.int64
    assert QueryTowerModule(5, 8, 16, layers=0).places.tolist() == [[0, 0]]
