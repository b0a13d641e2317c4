"""Layer norm of rows far from 0 on the GPU: a row's n comes from what it is apart from its mean, in both directions."""

import pytest
import torch

from tests import gpu_helpers as H
from tests import tower_oracle as O
from tests.test_gpu_tower import U, _data, _near

pytestmark = pytest.mark.gpu
st = torch.ops.st


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [7, 40, 1000, 1024, 4096, 5001, 18_000, 32_768])
def test_rows_of_one_value(dim, dtype):
    """n is 0 in both directions: the sums of a row's values are exact (24 bits hold them), and so is the mean.  The
    weight's gradient is 0, a row's r (g - mean g); 160 roundings of its terms, as for any row."""
    H.note(f"[tower] rows of one value {dim} {dtype}")
    values = torch.tensor([100.0, -1000.0, 3.25, 30_000.0 if dim <= 4096 else 30_720.0, 0.0])
    x = values.to(dtype).unsqueeze(1).repeat(1, dim)
    w, b, gy = _data((dim,), torch.float32, 2, 0.2, 1.0), _data((dim,), torch.float32, 3), _data((5, dim), dtype, 4, 1.0, 0.1)
    for eps in (1e-5, 1e-7):
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        y = st.layer_norm(*leaves, eps)
        assert torch.equal(y.detach().cpu(), b.to(dtype).expand(5, dim))
        gx, gw, _ = torch.autograd.grad(y, leaves, gy.cuda())
        assert not gw.any(), gw.abs().max()
        g, r = gy.double() * w.double(), eps ** -0.5
        mean = g.mean(1, keepdim=True)
        _near(gx, r * (g - mean), 160 * U * r * (g.abs() + g.abs().mean(1, keepdim=True)), "grad_x")
        # the sum of a residual of this type and x of zeros
        res = x.cuda().requires_grad_()
        y, total = st.dropout_add_layer_norm(torch.zeros_like(x).cuda(), res, leaves[1], leaves[2], 0.0, None, eps)
        gr, gw = torch.autograd.grad(y, [res, leaves[1]], gy.cuda())
        assert torch.equal(total.detach().cpu(), x) and torch.equal(gr, gx) and not gw.any()


def _steps_apart(rows, dim, dtype):
    """Rows of one value but for a few columns one step of 16 bits away; float32 ones spread by 2^-14 of their mean."""
    g = torch.Generator().manual_seed(dim)
    if dtype == torch.float32:
        return 4096.0 + 0.25 * torch.randn((rows, dim), generator=g)
    x = torch.full((rows, dim), 1000.0 if dtype == torch.float16 else 100.0)
    for row in x:
        row[torch.randperm(dim, generator=g)[:max(1, dim // 500)]] += 0.5
    return x.to(dtype)


def _terms(h, eps):
    """(n, r, c) in 64 bits, with the bounds where the 32-bit mean is off by e <= sigma / 8:

    with c = h - mean h and u = 2^-24, the differences from the 32-bit mean are c - e but for a rounding, and what their
    own mean (64 u of its magnitudes) takes back leaves u |c| + 66 u (mean |c| + e).  Their squares' sum less that mean's
    is off by 64 u (1 + e^2 / var) + 132 u e (mean |c| + e) / var < 90 u of itself, r by 50 u with its roundings.  So n is
    off by 70 u (|n| + mean |n| + e r).  e: 64 u A in float32, A = max |h|.  The 16-bit rows' sums are exact up to the
    joining of 16 waves (22 bits of 24), of u A each: 16 u A with the division's."""
    h = h.double()
    c = h - h.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    return c * r, r, c


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [24, 100, 201, 777, 1000, 4096, 5001, 16_000, 18_000, 24_576, 32_768])
def test_rows_of_values_steps_apart(dim, dtype):
    """What the mean's rounding leaves counts in every type, in both directions and in the codes."""
    H.note(f"[tower] rows steps apart {dim} {dtype}")
    rows, eps = 6, 1e-5
    x = _steps_apart(rows, dim, dtype)
    w, b, gy = _data((dim,), torch.float32, 2, 0.2, 1.0), _data((dim,), torch.float32, 3, 0.2, 0.0), _data((rows, dim), dtype, 4, 1.0, 0.1)
    n, r, c = _terms(x, eps)
    e = (64 if dtype == torch.float32 else 16) * U * x.double().abs().amax(1, keepdim=True)
    assert (e <= (c * c).mean(1, keepdim=True).sqrt() / 8).all()
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    dn = 70 * U * (n.abs() + mean(n.abs()) + e * r)
    dy = w.double().abs() * dn + 4 * U * ((n * w.double()).abs() + b.double().abs())
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = st.layer_norm(*leaves, eps)
    exact = [t.double().requires_grad_() for t in (x, w, b)]
    want = O.layer_norm(*exact, eps)
    _near(y, want, dy, "y")
    gx, gw, gb = torch.autograd.grad(y, leaves, gy.cuda())
    wx, ww, wb = torch.autograd.grad(want, exact, gy.double())
    g = gy.double() * w.double()
    _near(gx, wx, r * (160 * U * (g.abs() + mean(g.abs()) + n.abs() * mean((g * n).abs())) + dn * mean((g * n).abs())
                       + n.abs() * mean((g * dn).abs())), "grad_x")
    _near(gw, ww, ((64 + rows) * U * (gy.double() * n).abs() + gy.double().abs() * dn).sum(0), "grad_weight")
    _near(gb, wb, (64 + rows) * U * gy.double().abs().sum(0), "grad_bias")
    codes, scales = (t.cpu().double() for t in st.layer_norm_int8(x.cuda(), w.cuda(), b.cuda(), eps))
    most = want.detach().abs().amax(1)
    assert ((scales - most / 127).abs() <= dy.amax(1) / 127 + 2 * U * most / 127).all()
    s = scales.unsqueeze(1)
    assert ((codes[:, :dim] - want.detach() / s).abs() <= 0.5 + dy / s + 127 * 4 * U).all()
