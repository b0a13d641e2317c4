"""The query tower's operators where offsets pass 32 bits: the last rows are those of a small call on them alone, and the
first.  Kept elements, codes and the sums of a row do not depend on the call's size, so the bits are equal."""

import numpy as np
import pytest
import torch

from tests import gpu_helpers as H
from tests import tower_oracle as O

pytestmark = pytest.mark.gpu
st = torch.ops.st


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _rows(rows, dim, dtype):
    """Rows that repeat 10,007 drawn ones, so that those at the end differ from those at the start."""
    some = torch.randn((10_007, dim), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    return some[torch.arange(rows, device="cuda") % 10_007]


def test_layer_norm_past_32_bits():
    H.note("[tower] layer_norm of 2.2e9 elements")
    rows, dim = 2_150_000, 1024
    x = _rows(rows, dim, torch.bfloat16).requires_grad_()
    w, b = (torch.randn(dim, generator=torch.Generator().manual_seed(k)).cuda() for k in (2, 3))
    y = st.layer_norm(x, w, b)
    gy = y.detach()
    gx, = torch.autograd.grad(y, x, gy)
    for part in (slice(0, 70), slice(rows - 70, rows)):
        leaf = x.detach()[part].clone().requires_grad_()
        small = st.layer_norm(leaf, w, b)
        assert torch.equal(gy[part], small)
        assert torch.equal(gx[part], torch.autograd.grad(small, leaf, small.detach())[0])


def test_dropout_past_32_bits():
    H.note("[tower] dropout of 4.4e9 elements")
    n = (1 << 32) + 100_003
    state = [3, 1 << 40]
    y = st.dropout(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.5, torch.tensor(state).cuda())
    first = n - 50_003
    assert first % 8 == 0
    blocks = np.arange(first // 8, (n + 7) // 8, dtype=np.uint64)
    whole = np.zeros_like(blocks)
    words = O.philox([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), whole, whole + np.uint64(1 << 8)], [3, 0])
    halves = np.stack([h for v in words for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], 1).reshape(-1)
    assert torch.equal((y[first:] != 0).cpu(), torch.from_numpy(halves[:n - first] >= 1 << 15))


def test_int8_past_32_bits():
    """A table of 4.6e9 bytes, results past 2^32 bytes, vectors past 2^31 elements."""
    H.note("[tower] int8 table of 4.6e9 bytes")
    rows, dim = 36_000_003, 128
    table, scales = st.int8_quantize(_rows(rows, dim, torch.float16))
    x = _rows(33, dim, torch.float32)
    for tokens in (1, 33):
        y = st.int8_matmul(table, scales, x[:tokens])
        for part in (slice(0, 300), slice(rows - 300, rows)):
            assert torch.equal(y[:, part], st.int8_matmul(table[part].clone(), scales[part].clone(), x[:tokens]))
    del table, scales, y
    torch.cuda.empty_cache()
    many = _rows(2_200_000, 1024, torch.bfloat16)
    codes, code_scales = st.int8_quantize(many)
    small, small_scales = st.int8_quantize(many[-70:])
    assert torch.equal(codes[-70:], small) and torch.equal(code_scales[-70:], small_scales)
    weight, weight_scales = st.int8_quantize(_rows(140, 1024, torch.float32))
    y = st.int8_matmul(weight, weight_scales, many, None, None, torch.bfloat16)
    assert torch.equal(y[-70:], st.int8_matmul(weight, weight_scales, many[-70:], None, None, torch.bfloat16))
