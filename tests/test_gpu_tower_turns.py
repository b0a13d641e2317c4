"""Layer norm, alone and of a residual plus dropout, over more rows than the chip's
workgroups take at once: every row and every gradient against 64 bits.

The plain forms run on the GPU in float64; dropout's numbers come from
tests/tower_oracle.py.  Bounds are those of test_gpu_tower_offsets.py (u = 2^-24,
A = max |h|, e = 64 u A, r = 1 / sqrt(var + eps)): n is off by dn = 70 u (|n| +
mean |n| + e r).  The weight's and the bias's gradients go through at most 128
additions each here, not one a row: of a lane's rows (at most 16), of a
workgroup's (64), of the parts that a thread takes (at most 32), ten in a tree."""

import functools

import pytest
import torch

from tests import gpu_helpers as H
from tests import tower_oracle as O
from tests.test_gpu_tower import HALF, TINY, U

pytestmark = pytest.mark.gpu
st = torch.ops.st
EPS, P, STATE = 1e-5, 0.3, (1 << 40) + 7


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _within(got, want, atol, what):
    atol = atol + HALF[got.dtype] * (want.abs() + atol) + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert (off <= atol).all(), (what, int((off > atol).sum()), (off / atol).max().item())


def _draw(shape, dtype, seed, scale=1.0, shift=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


@functools.lru_cache(maxsize=1)
def _keeps(rows, dim):
    return O.keeps((rows, dim), P, (STATE, 5)).cuda()


def _check(h, w, b, y, gy, gsum, keep, grads):
    """y and the gradients (x, residual or None, weight, bias) of the norm of rows h."""
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    h64, w64, b64, g64 = h.double(), w.detach().double(), b.detach().double(), gy.double()
    c = h64 - mean(h64)
    r = 1 / torch.sqrt(mean(c * c) + EPS)
    n = c * r
    dn = 70 * U * (n.abs() + mean(n.abs()) + 64 * U * h64.abs().amax(1, keepdim=True) * r)
    _within(y.detach(), n * w64 + b64, w64.abs() * dn + 4 * U * ((n * w64).abs() + b64.abs()), "y")
    g = g64 * w64
    gh = r * (g - mean(g) - n * mean(g * n))
    bound = r * (160 * U * (g.abs() + mean(g.abs()) + n.abs() * mean((g * n).abs())) + dn * mean((g * n).abs())
                 + n.abs() * mean((g * dn).abs()))
    if gsum is not None:
        gh = gh + gsum.double()
        bound = bound + U * (gsum.double().abs() + gh.abs())
        _within(grads[1], gh, bound, "grad_residual")
    if keep is not None:
        stay = keep.double() * O.times(P)
        gh, bound = gh * stay, bound * stay * (1 + 2 * U) + 2 * U * (gh * stay).abs()
    _within(grads[0], gh, bound, "grad_x")
    _within(grads[2], (g64 * n).sum(0), (128 * U * (g64 * n).abs() + g64.abs() * dn).sum(0), "grad_weight")
    _within(grads[3], g64.sum(0), 128 * U * g64.abs().sum(0), "grad_bias")


@pytest.mark.parametrize("dtype,residual_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                 (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                                 (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,dim", [(150_001, 64), (40_003, 200), (10_007, 777), (5003, 2048), (2503, 5001), (1203, 12_000),
                                      (701, 17_001), (701, 20_000), (601, 32_768)])
def test_rows_in_turns(rows, dim, dtype, residual_type):
    H.note(f"[tower] in turns {rows} x {dim} {dtype} {residual_type}")
    x, res = _draw((rows, dim), dtype, 1, 1.5, 0.3), _draw((rows, dim), residual_type, 2, 2.0, -0.1)
    gy, gs = _draw((rows, dim), dtype, 3), _draw((rows, dim), residual_type, 4, 0.7)
    w, b = (_draw((dim,), torch.float32, 5, 0.2, 1.0).requires_grad_(), _draw((dim,), torch.float32, 6, 0.2).requires_grad_())
    leaf = x.clone().requires_grad_()
    if residual_type == dtype:
        y = st.layer_norm(leaf, w, b, EPS)
        gx, gw, gb = torch.autograd.grad(y, [leaf, w, b], gy)
        _check(x, w, b, y, gy, None, None, (gx, None, gw, gb))
    keep, other = _keeps(rows, dim), res.clone().requires_grad_()
    y, total = st.dropout_add_layer_norm(leaf, other, w, b, P, torch.tensor([STATE, 5]).cuda(), EPS)
    held = (res.float() + torch.where(keep, x.float() * torch.tensor(O.times(P), dtype=torch.float32).cuda(), 0.0)).to(residual_type)
    assert torch.equal(total.detach(), held)
    grads = torch.autograd.grad([y, total], [leaf, other, w, b], [gy, gs])
    _check(held, w, b, y, gy, gs, keep, grads)
