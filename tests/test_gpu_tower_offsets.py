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
