"""The query tower's operators on the GPU against plain forms
(tests/tower_oracle.py): layer norm, dropout, their sum with a residual, rows
in 8 bits and their products; gradients against 64 bits and differences.

Tolerances (u = 2^-24, the rounding of 32 bits; `HALF` a half unit of the
result's type; A = max |h| of a row, r = 1 / sqrt(var + eps)):
- a row's sums have at most 32 terms a lane, then a tree of ten: relative 42 u
  of the sum of magnitudes, 64 u with the product by 1 / columns and roundings.
  The mean is off by 64 u A, n by dn = r 64 u A + 70 u |n| (a shift of the mean
  enters the variance by its square), y by |w| dn + 4 u (|n w| + |b|).
- gh = r (g - mean g - n mean(g n)): 160 u of the sum of its terms' magnitudes,
  r dn mean |g n| of its own n and r |n| mean |g dn| of the others'.
- gw = sum gy n over rows: (64 + rows) u of the sum of magnitudes, and sum |gy| dn.
- dropout, the sum with a residual and the codes of rows are single roundings in
  a stated order: equal bits.
- an 8-bit product's sum is exact; its conversion, two products and the bias's
  addition are four roundings: 5 u (|y| + |bias|), then one to its type.
"""

import math
import threading

import pytest
import torch

from tests import gpu_helpers as H
from tests import tower_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
st = torch.ops.st


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _near(got, want, atol, what=""):
    """got within atol of want before its rounding to got's type; values that are not finite, or past it, are the same."""
    want = want.detach().double()
    want = torch.where(want.abs() > torch.finfo(got.dtype).max, want.sign() * math.inf, want)
    atol = torch.as_tensor(atol, dtype=torch.float64).expand(want.shape)
    atol = atol + HALF[got.dtype] * (want.abs() + atol) + TINY[got.dtype]
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), what
    off = (got - want).abs()
    bad = fine & ~(off <= atol)
    assert not bad.any(), (what, int(bad.sum()), off[bad][:5], atol[bad][:5], want[bad][:5])


def _state(seed):
    return torch.randint(-(1 << 63), (1 << 63) - 1, (2,), generator=torch.Generator().manual_seed(seed))


def _data(shape, dtype, seed, scale=1.5, shift=0.3):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale + shift).to(dtype)


# ------------------------------------------------------------------ dropout


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 7), (1, 2048), (2049,), (33, 1001), (0, 5), ()])
def test_dropout(shape, dtype):
    """Kept elements times the factor, rounded once, 0 elsewhere, in both directions; the state may advance in between."""
    H.note(f"[tower] dropout {shape} {dtype}")
    for p in (0.0, 0.1, 0.5, 0.937, 1.0):
        state = _state(7)
        x, g = _data(shape, dtype, 1), _data(shape, dtype, 2)
        leaf, moving = x.cuda().requires_grad_(), state.cuda()
        y = st.dropout(leaf, p, moving)
        moving += 1
        grad, = torch.autograd.grad(y, leaf, g.cuda())
        if x.numel():
            assert torch.equal(y.detach().cpu(), O.dropped(x, p, state).to(dtype))
            assert torch.equal(grad.cpu(), O.dropped(g, p, state).to(dtype))
        assert y.shape == x.shape and grad.dtype == dtype
        assert torch.equal(st.dropout(x.cuda(), p, state.cuda()), y.detach())


def test_dropout_layouts_and_values():
    """Elements count in the tensor's order, whatever its strides; what a dropped element holds does not matter."""
    H.note("[tower] dropout layouts")
    state = _state(11)
    x = _data((40, 24), torch.float32, 3)
    want = O.dropped(x, 0.4, state)
    for t in (x.cuda(), x.cuda().t().contiguous().t(), torch.nn.functional.pad(x, (3, 2)).cuda()[:, 3:27],
              torch.cat([torch.zeros(1), x.flatten()]).cuda()[1:].view(40, 24)):
        assert torch.equal(st.dropout(t, 0.4, state.cuda()).cpu(), want)
    assert torch.equal(st.dropout(x, 0.4, state), want)  # CPU tensors
    stay = O.keeps(x.shape, 0.4, state)
    odd = torch.where(stay, x, torch.tensor([math.nan, math.inf, -math.inf]).repeat(320).view(40, 24))
    assert torch.equal(st.dropout(odd.cuda(), 0.4, state.cuda()).cpu(), want)
    grown = torch.full((16,), 60_000.0, dtype=torch.float16)
    assert torch.equal(st.dropout(grown.cuda(), 0.5, state.cuda()).cpu(), O.dropped(grown, 0.5, state).half())
    # the gradient of a sum is one element, expanded
    leaf = x.cuda().requires_grad_()
    st.dropout(leaf, 0.4, state.cuda()).sum().backward()
    assert torch.equal(leaf.grad.cpu(), O.dropped(torch.ones_like(x), 0.4, state))
    # other states, other elements
    other = state.clone()
    other[1] += 1
    assert not torch.equal(O.keeps(x.shape, 0.4, other), stay)
    assert torch.equal(st.dropout(x.cuda(), 0.4, other.cuda()).cpu(), O.dropped(x, 0.4, other))


def test_dropout_large():
    """More workgroups than the chip holds; the last elements are right too."""
    H.note("[tower] dropout large")
    n = (1 << 26) + 5
    state = _state(5)
    y = st.dropout(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.25, state.cuda())
    stay = O.keeps((n,), 0.25, state)
    assert torch.equal((y != 0).cpu(), stay)
    assert set(y.unique().tolist()) == {0.0, torch.tensor(4 / 3).bfloat16().item()}


# ------------------------------------------------------------------ layer norm


def _norm_terms(h, w, b, eps):
    """(n, r, dn) of rows h in 64 bits and the bound of y."""
    h = h.double()
    centred = h - h.mean(1, keepdim=True)
    r = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + eps)
    n = centred * r
    dn = r * 64 * U * h.abs().amax(1, keepdim=True) + 70 * U * n.abs()
    return n, r, dn, w.abs() * dn + 4 * U * ((n * w).abs() + b.abs())


def _check_gradients(h, w, gy, gsum, got, want, eps, p=0.0, state=None):
    """got: the gradients (x, residual or None, weight, bias) with their types; want: the same in 64 bits."""
    n, r, dn, _ = _norm_terms(h, w, torch.zeros_like(w), eps)
    gy = gy.double()
    g = gy * w
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    bound = r * (160 * U * (g.abs() + mean(g.abs()) + n.abs() * mean((g * n).abs())) + dn * mean((g * n).abs())
                 + n.abs() * mean((g * dn).abs()))
    if gsum is not None:
        bound = bound + U * (gsum.double().abs() + want[1].abs() if want[1] is not None else 0.0)
    if got[1] is not None:
        _near(got[1], want[1], bound, "grad_residual")
    if got[0] is not None:
        stay = O.keeps(h.shape, p, state).double() * O.times(p) * (1 + 2 * U) if p else 1.0
        _near(got[0], want[0], bound * stay + (2 * U * want[0].abs() if p else 0.0), "grad_x")
    rows = len(h)
    _near(got[2], want[2], ((64 + rows) * U * (gy * n).abs() + gy.abs() * dn).sum(0), "grad_weight")
    _near(got[3], want[3], (64 + rows) * U * gy.abs().sum(0), "grad_bias")


SIZES = [(1, 1), (5, 2), (3, 7), (9, 8), (33, 63), (31, 64), (17, 65), (70, 128), (65, 129), (40, 255), (5, 256), (12, 257),
         (9, 511), (6, 512), (301, 513), (8, 1000), (7, 1024), (5, 1025), (4, 2047), (3, 2048), (9, 2049), (2, 4096),
         (3, 5003), (2, 8192), (2, 8193), (1, 16_384), (3, 16_385), (2, 32_767), (2, 32_768)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", SIZES)
def test_layer_norm(rows, dim, dtype):
    H.note(f"[tower] layer_norm {rows} x {dim} {dtype}")
    for weights in {dtype, torch.float32}:
        x, w, b = _data((rows, dim), dtype, rows + dim), _data((dim,), weights, 2, 0.2, 1.0), _data((dim,), weights, 3, 0.2, 0.0)
        gy = _data((rows, dim), dtype, 4, 1.0, 0.1)
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        y = st.layer_norm(*leaves, 1e-5)
        assert y.dtype == dtype
        grads = torch.autograd.grad(y, leaves, gy.cuda())
        exact = [t.double().requires_grad_() for t in (x, w, b)]
        want = O.layer_norm(*exact)
        _near(y, want, _norm_terms(x, w.double(), b.double(), 1e-5)[3], "y")
        gx, gw, gb = torch.autograd.grad(want, exact, gy.double())
        assert [g.dtype for g in grads] == [dtype, weights, weights]
        _check_gradients(x, w.double(), gy, None, (grads[0], None, *grads[1:]), (gx, None, gw, gb), 1e-5)
        with torch.no_grad():
            assert torch.equal(st.layer_norm(*leaves, 1e-5), y)


@pytest.mark.parametrize("rows,dim", [(10_007, 64), (5001, 200), (3000, 1024), (1500, 2100)])
def test_layer_norm_many_rows(rows, dim):
    """More rows than the chip's workgroups take at once."""
    H.note(f"[tower] layer_norm {rows} x {dim}")
    x, w, b = _data((rows, dim), torch.bfloat16, 1), _data((dim,), torch.float32, 2, 0.2, 1.0), _data((dim,), torch.float32, 3)
    gy = _data((rows, dim), torch.bfloat16, 4, 1.0, 0.1)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = st.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, gy.cuda())
    exact = [t.double().requires_grad_() for t in (x, w, b)]
    want = O.layer_norm(*exact)
    _near(y, want, _norm_terms(x, w.double(), b.double(), 1e-5)[3], "y")
    gx, gw, gb = torch.autograd.grad(want, exact, gy.double())
    _check_gradients(x, w.double(), gy, None, (grads[0], None, *grads[1:]), (gx, None, gw, gb), 1e-5)
    # the same bits every time
    again = torch.autograd.grad(st.layer_norm(*leaves), leaves, gy.cuda())
    assert all(torch.equal(a, c) for a, c in zip(grads, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(70_001, 20), (90_001, 100), (40_003, 201), (9001, 1001), (3001, 5004), (1201, 16_001),
                                      (1201, 17_001), (1201, 24_576), (1101, 25_001), (1101, 32_768)])
def test_layer_norm_rows_in_turns(rows, dim, dtype):
    """Rows that a workgroup takes one after another have the bits of rows in calls of their own; the bias's gradient is
    the sum of the parts' (the whole and all parts are off by 64 + rows roundings of the magnitudes each at most)."""
    H.note(f"[tower] layer_norm in turns {rows} x {dim} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(dim)
    x, gy = (torch.randn((rows, dim), generator=g, device="cuda").to(dtype) for _ in range(2))
    res = torch.randn((rows, dim), generator=g, device="cuda").to(dtype)
    w, b = (torch.randn(dim, generator=g, device="cuda").requires_grad_() for _ in range(2))

    def both(part):
        leaves = [x[part].detach().requires_grad_(), res[part].detach().requires_grad_()]
        y = st.layer_norm(leaves[0], w, b)
        z, total = st.dropout_add_layer_norm(*leaves, w, b)
        grads = torch.autograd.grad(y, [leaves[0], w, b], gy[part])
        more = torch.autograd.grad([z, total], leaves, [gy[part], gy[part]])
        codes = st.layer_norm_int8(x[part], w.detach(), b.detach()) + st.int8_quantize(x[part])
        return [y.detach(), z.detach(), total.detach(), grads[0], *more, *codes], grads[1:]

    whole, sums = both(slice(0, rows))
    step = 128
    parts = [both(slice(at, min(at + step, rows))) for at in range(0, min(rows, 10 * step), step)]
    parts.append(both(slice(rows - 37, rows)))
    ends = [(at, min(at + step, rows)) for at in range(0, min(rows, 10 * step), step)] + [(rows - 37, rows)]
    for (lo, hi), (own, _) in zip(ends, parts):
        for i, (a, c) in enumerate(zip(whole, own)):
            assert torch.equal(a[lo:hi], c), (i, lo)
    if rows <= 10 * step:
        magnitude = gy.double().abs().sum(0)
        total = sum(p[1][1].double() for p in parts[:-1])
        assert ((sums[1].double() - total).abs() <= 2 * (64 + rows) * U * magnitude).all()


def test_layer_norm_forms():
    """Without weight or bias, of any shape and stride, no rows, one wanted gradient, CPU tensors."""
    H.note("[tower] layer_norm forms")
    x, w, b = _data((6, 5, 40), torch.float32, 1), _data((40,), torch.float32, 2, 0.2, 1.0), _data((40,), torch.float32, 3)
    flat = x.view(30, 40)
    one, zero = torch.ones(40), torch.zeros(40)
    for weight, bias in ((None, None), (w, None), (None, b), (w, b)):
        y = st.layer_norm(x.cuda(), *(t.cuda() if t is not None else None for t in (weight, bias)))
        bound = _norm_terms(flat, (one if weight is None else weight).double(), (zero if bias is None else bias).double(), 1e-5)[3]
        _near(y.view(30, 40), O.layer_norm(flat.double(), weight, bias), bound)
        assert torch.equal(st.layer_norm(x, weight, bias), y.cpu())
        leaf = x.cuda().requires_grad_()
        st.layer_norm(leaf, *(t.cuda() if t is not None else None for t in (weight, bias))).square().sum().backward()
        assert leaf.grad.shape == x.shape
    want = st.layer_norm(flat.cuda(), w.cuda(), b.cuda())
    wide = torch.nn.functional.pad(flat, (3, 6), value=math.nan).cuda()[:, 3:43]
    assert torch.equal(st.layer_norm(wide, w.cuda(), b.cuda()), want)
    assert torch.equal(st.layer_norm(flat.cuda().t().contiguous().t(), w.cuda(), b.cuda()), want)
    assert torch.equal(st.layer_norm(flat.cuda()[4], w.cuda(), b.cuda()), want[4])
    assert torch.equal(st.layer_norm(flat.cuda()[3].expand(7, 40), w.cuda(), b.cuda()), want[3].expand(7, 40))
    assert torch.equal(st.layer_norm(flat.cuda(), torch.stack([w, w], 1).cuda()[:, 0], b.cuda()), want)
    # gradients through strides, and on the CPU
    gy = _data((30, 40), torch.float32, 5).cuda()
    a, c = wide.detach().requires_grad_(), flat.cuda().requires_grad_()
    assert torch.equal(torch.autograd.grad(st.layer_norm(a, w.cuda()), a, gy)[0],
                       torch.autograd.grad(st.layer_norm(c, w.cuda()), c, gy.t().contiguous().t())[0])
    host = [t.clone().requires_grad_() for t in (flat, w, b)]
    there = [t.cuda().requires_grad_() for t in (flat, w, b)]
    for g, k in zip(torch.autograd.grad(st.layer_norm(*host), host, gy.cpu()), torch.autograd.grad(st.layer_norm(*there), there, gy)):
        assert g.device.type == "cpu" and torch.equal(g, k.cpu())
    # only the bias's gradient
    only = b.cuda().requires_grad_()
    assert torch.equal(torch.autograd.grad(st.layer_norm(flat.cuda(), w.cuda(), only), only, gy)[0],
                       torch.autograd.grad(st.layer_norm(*there), there, gy)[2])
    # no rows
    none = [torch.zeros((0, 40), device="cuda").requires_grad_(), *there[1:]]
    y = st.layer_norm(*none)
    gx, gw, gb = torch.autograd.grad(y, none, torch.zeros_like(y))
    assert gx.shape == (0, 40) and not gw.any() and not gb.any()


def test_layer_norm_values():
    """Rows of one value, of large offsets and scales, and rows that are not finite, which leave the others alone."""
    H.note("[tower] layer_norm values")
    x = _data((8, 300), torch.float32, 1)
    x[1] = 3.25
    x[2] += 4096.0
    x[3] *= 2.0 ** 50
    x[4] *= 2.0 ** -60
    x[5, 7] = math.nan
    x[6, 100] = math.inf
    y = st.layer_norm(x.cuda(), None, None, 1e-5).cpu()
    fine = [0, 1, 2, 3, 4, 7]
    one = torch.ones(300, dtype=torch.float64)
    _near(y[fine], O.layer_norm(x[fine].double()), _norm_terms(x[fine], one, 0 * one, 1e-5)[3])
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all()
    assert not y[1].any()


def test_layer_norm_gradient_against_differences():
    H.note("[tower] layer_norm differences")
    x, w, b = _data((4, 37), torch.float32, 1), _data((37,), torch.float32, 2, 0.2, 1.0), _data((37,), torch.float32, 3)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    gy = _data((4, 37), torch.float32, 5)
    grads = torch.autograd.grad(st.layer_norm(*leaves), leaves, gy.cuda())
    f = lambda *t: (O.layer_norm(*t) * gy.double()).sum()  # noqa: E731
    at = [t.double() for t in (x, w, b)]
    g = torch.Generator().manual_seed(9)
    for i, grad in enumerate(grads):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        step = lambda s: f(*[t + s * 1e-4 * d if k == i else t for k, t in enumerate(at)])  # noqa: E731
        slope = (step(1) - step(-1)) / 2e-4
        # central differences are off by the third derivative times 1e-8 / 6; 1e-5 of the terms' size holds both
        size = (grad.cpu().double() * d).abs().sum()
        assert abs((grad.cpu().double() * d).sum() - slope) < 1e-5 * size


# ------------------------------------------------------------------ dropout, residual and norm in one


@pytest.mark.parametrize("dtype,residual_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                 (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                                 (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (33, 64), (17, 65), (20, 128), (9, 255), (4, 512), (301, 513), (5, 1001),
                                      (3, 2048), (2, 2500), (3, 4097), (2, 16_000), (2, 20_001)])
def test_dropout_add_layer_norm(rows, dim, dtype, residual_type):
    """The sum has the bits of residual + dropout(x); the norm is the sum's; all five gradients."""
    H.note(f"[tower] dropout_add_layer_norm {rows} x {dim} {dtype} {residual_type}")
    for p in (0.0, 0.3):
        state = _state(rows + dim)
        x, res = _data((rows, dim), dtype, 1), _data((rows, dim), residual_type, 2, 2.0, -0.1)
        w, b = _data((dim,), torch.float32, 3, 0.2, 1.0), _data((dim,), torch.float32, 4, 0.2, 0.0)
        gy, gs = _data((rows, dim), dtype, 5, 1.0, 0.1), _data((rows, dim), residual_type, 6, 0.7, 0.0)
        leaves = [t.cuda().requires_grad_() for t in (x, res, w, b)]
        moving = state.cuda()
        y, total = st.dropout_add_layer_norm(*leaves, p, moving)
        moving += 3
        held = (res.float() + (O.dropped(x, p, state) if p else x.float())).to(residual_type)
        assert torch.equal(total.detach().cpu(), held) and y.dtype == dtype
        exact = [t.double().requires_grad_() for t in (held, w, b)]
        want = O.layer_norm(*exact)
        _near(y, want, _norm_terms(held, w.double(), b.double(), 1e-5)[3], "y")
        gh, gw, gb = torch.autograd.grad(want, exact, gy.double())
        gh = gh + gs.double()
        gx = torch.where(O.keeps(x.shape, p, state), gh * O.times(p), 0.0) if p else gh
        grads = torch.autograd.grad([y, total], leaves, [gy.cuda(), gs.cuda()])
        assert [g.dtype for g in grads] == [dtype, residual_type, torch.float32, torch.float32]
        _check_gradients(held, w.double(), gy, gs, grads, (gx, gh, gw, gb), 1e-5, p, state)


@pytest.mark.parametrize("dtype,residual_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                 (torch.float16, torch.float32)])
@pytest.mark.parametrize("dim", [10, 16, 20, 24, 30, 32, 41, 48, 90, 96, 180, 370, 384, 750, 768, 1500, 1536, 6000, 12_000])
def test_dropout_add_layer_norm_of_whole_and_ragged_rows(dim, dtype, residual_type):
    """Lanes whose last step of columns is whole, in part or empty, in workgroups of many rows and of one."""
    test_dropout_add_layer_norm(37, dim, dtype, residual_type)


def test_two_threads_at_once():
    """Passes of two threads on streams of their own give the bits that they give alone."""
    H.note("[tower] two threads")
    w = _data((900,), torch.float32, 3, 0.2, 1.0).cuda()
    table, scales, _ = (t.cuda() for t in _table(700, 900, 1))

    def step(seed):
        x, res = (_data((400, 900), torch.bfloat16, seed + i).cuda().requires_grad_() for i in range(2))
        own = w.clone().requires_grad_()
        y, total = st.dropout_add_layer_norm(x, res, own, None, 0.2, _state(seed).cuda())
        grads = torch.autograd.grad([y, total], [x, res, own], [x.detach(), res.detach()])
        return [y.detach(), total.detach(), *grads, st.int8_matmul(table, scales, x.detach()),
                st.int8_matmul(table, scales, x.detach()[:2])]

    alone = [[step(10 * k + i) for i in range(4)] for k in range(2)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[k] = [step(10 * k + i) for i in range(4)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(alone, got):
        for c, d in zip(a, b):
            assert all(torch.equal(p, q) for p, q in zip(c, d))


def test_dropout_add_layer_norm_forms():
    """One gradient of the two results, of the two inputs; strides; shapes; the same numbers as dropout's."""
    H.note("[tower] dropout_add_layer_norm forms")
    state = _state(3)
    x, res = _data((4, 6, 72), torch.float32, 1), _data((4, 6, 72), torch.float32, 2)
    w = _data((72,), torch.float32, 3, 0.2, 1.0).cuda()
    y, total = st.dropout_add_layer_norm(x.cuda(), res.cuda(), w, None, 0.5, state.cuda())
    assert y.shape == total.shape == x.shape
    assert torch.equal(total, res.cuda() + st.dropout(x.cuda(), 0.5, state.cuda()))
    assert torch.equal(y, st.layer_norm(total, w))
    host = st.dropout_add_layer_norm(x, res, w.cpu(), None, 0.5, state)
    assert torch.equal(host[0], y.cpu()) and torch.equal(host[1], total.cpu())
    flat = lambda t: torch.nn.functional.pad(t.view(24, 72), (1, 4), value=math.nan).cuda()[:, 1:73]  # noqa: E731
    again = st.dropout_add_layer_norm(flat(x), flat(res), w, None, 0.5, state.cuda())
    assert torch.equal(again[0].view_as(y), y) and torch.equal(again[1].view_as(y), total)
    gy, gs = _data(x.shape, torch.float32, 5).cuda(), _data(x.shape, torch.float32, 6).cuda()
    a, c = x.cuda().requires_grad_(), res.cuda().requires_grad_()

    def grads(outs, given, leaves):
        o = st.dropout_add_layer_norm(a, c, w, None, 0.5, state.cuda())
        return torch.autograd.grad([o[i] for i in outs], leaves, given)

    both = grads([0, 1], [gy, gs], [a, c])
    zero = torch.zeros_like(gy)
    assert all(torch.equal(i, k) for i, k in zip(grads([0], [gy], [a, c]), grads([0, 1], [gy, zero], [a, c])))
    assert all(torch.equal(i, k) for i, k in zip(grads([1], [gs], [a, c]), grads([0, 1], [zero, gs], [a, c])))
    assert torch.equal(grads([1], [gs], [c])[0], gs)
    assert torch.equal(grads([0, 1], [gy, gs], [a])[0], both[0]) and torch.equal(grads([0, 1], [gy, gs], [c])[0], both[1])
    # what a dropped element holds does not matter
    stay = O.keeps(x.shape, 0.5, state)
    odd = torch.where(stay, x, math.nan)
    assert torch.equal(st.dropout_add_layer_norm(odd.cuda(), res.cuda(), w, None, 0.5, state.cuda())[0], y)


# ------------------------------------------------------------------ rows in 8 bits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 15), (7, 16), (33, 17), (9, 128), (20, 200), (4, 513), (3, 1025), (9, 2049),
                                      (2, 5000), (3, 9001), (2, 32_768), (3, 32_769), (2, 100_001)])
def test_int8_quantize(rows, dim, dtype):
    H.note(f"[tower] int8_quantize {rows} x {dim} {dtype}")
    x = _data((rows, dim), dtype, rows * dim)
    x[0] *= 2.0 ** -10
    codes, scales = st.int8_quantize(x.cuda())
    want, want_scales = O.codes(x)
    assert codes.dtype == torch.int8 and torch.equal(codes.cpu(), want)
    assert torch.equal(scales.cpu(), want_scales)
    host = st.int8_quantize(x)
    assert torch.equal(host[0], want) and torch.equal(host[1], want_scales)


@pytest.mark.parametrize("dim", [40, 40_000])
def test_int8_quantize_values(dim):
    """Rows of zeros, of values below 2^-119, of halves between codes; rows that are not finite; strides; no rows."""
    H.note(f"[tower] int8_quantize values {dim}")
    x = _data((8, dim), torch.float32, 1)
    x[0] = 0.0
    x[1] = 2.0 ** -120
    x[2] = torch.arange(dim) % 255 - 127 + 0.5
    x[2, 0] = 127.0
    x[3, 5] = math.nan
    x[4, 6] = -math.inf
    x[5] *= 2.0 ** 100
    x[6] = -x[6].abs()
    codes, scales = st.int8_quantize(x.cuda())
    want, want_scales = O.codes(x)
    assert torch.equal(codes.cpu(), want)
    assert torch.equal(torch.isnan(scales.cpu()), torch.isnan(want_scales))
    assert torch.equal(scales.cpu().nan_to_num(7.0), want_scales.nan_to_num(7.0))
    wide = torch.nn.functional.pad(x, (1, 2), value=9e9).cuda()[:, 1:-2]
    assert torch.equal(st.int8_quantize(wide)[0].cpu(), want)
    deep = st.int8_quantize(x.view(2, 4, dim).cuda())
    assert deep[0].shape == (2, 4, want.shape[1]) and deep[1].shape == (2, 4) and torch.equal(deep[0].view_as(want).cpu(), want)
    assert st.int8_quantize(x[0].cuda())[1].shape == ()
    none = st.int8_quantize(x[:0].cuda())
    assert none[0].shape == (0, want.shape[1]) and none[1].shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 17), (33, 64), (9, 250), (3, 512), (5, 1024), (3, 3000), (2, 8000), (2, 20_000)])
def test_layer_norm_int8(rows, dim, dtype):
    """The codes of the norm's 32-bit values: equal to the 64-bit norm's but where it lies near a half."""
    H.note(f"[tower] layer_norm_int8 {rows} x {dim} {dtype}")
    x, w, b = _data((rows, dim), dtype, 1), _data((dim,), torch.float32, 2, 0.2, 1.0), _data((dim,), torch.float32, 3, 0.2, 0.0)
    codes, scales = st.layer_norm_int8(x.cuda(), w.cuda(), b.cuda())
    y = O.layer_norm(x.double(), w.double(), b.double())
    bound = _norm_terms(x, w.double(), b.double(), 1e-5)[3]
    most = y.abs().amax(1)
    assert ((scales.cpu().double() - most / 127).abs() <= bound.amax(1) / 127 + 2 * U * most / 127).all()
    assert not codes[:, dim:].any()
    q = y / scales.cpu().double().unsqueeze(1)
    off = (codes[:, :dim].cpu().double() - q).abs()
    assert (off <= 0.5 + bound / scales.cpu().double().unsqueeze(1) + 127 * 4 * U).all()
    assert all(torch.equal(a, c.cpu()) for a, c in zip(st.layer_norm_int8(x, w, b), (codes, scales)))


def _table(rows, dim, seed):
    g = torch.Generator().manual_seed(seed)
    columns = -(-dim // 16) * 16
    codes = torch.randint(-128, 128, (rows, columns), generator=g, dtype=torch.int8)
    return codes, torch.rand(rows, generator=g) + 0.1, torch.randn(rows, generator=g)


def _check_matmul(table, scales, x, x_scales, bias, out, cuda_x=None, cuda_scales=None):
    """x: codes and scales that the product has to give the sums of; cuda_x: what is passed (x itself without it)."""
    want = O.matmul(table, scales, x, x_scales, bias)
    got = st.int8_matmul(table.cuda(), scales.cuda(), x.cuda() if cuda_x is None else cuda_x,
                         x_scales.cuda() if cuda_x is None else cuda_scales, None if bias is None else bias.cuda(), out)
    assert got.dtype == (out or got.dtype)
    size = (want if bias is None else want - bias.double()).abs() + (0.0 if bias is None else bias.double().abs())
    _near(got, want, 5 * U * size, "y")
    return got


@pytest.mark.parametrize("tokens", [1, 2, 4, 15, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("rows,dim", [(1, 16), (5, 48), (63, 64), (64, 100), (65, 128), (300, 200), (1000, 1024), (257, 1040),
                                      (130, 2064)])
def test_int8_matmul(tokens, rows, dim):
    H.note(f"[tower] int8_matmul {tokens} x {dim} x {rows}")
    table, scales, bias = _table(rows, dim, tokens + rows)
    if dim % 16 == 0:
        x, x_scales, _ = _table(tokens, dim, tokens)
        _check_matmul(table, scales, x, x_scales, None, None)
        _check_matmul(table, scales, x, x_scales, bias, torch.bfloat16)
    for dtype, out in ((torch.float32, None), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)):
        x = _data((tokens, dim), dtype, dim)
        _check_matmul(table, scales, *O.codes(x), bias if dtype == torch.float16 else None, out, x.cuda())


@pytest.mark.parametrize("tokens,rows,dim", [(1, 200_000, 64), (3, 150_001, 144), (40, 140_000, 256), (70, 9000, 512),
                                             (300, 1000, 300), (513, 777, 1500), (1025, 515, 4112), (2, 8200, 8192)])
def test_int8_matmul_large(tokens, rows, dim):
    H.note(f"[tower] int8_matmul {tokens} x {dim} x {rows}")
    table, scales, bias = _table(rows, dim, 1)
    x = _data((tokens, dim), torch.bfloat16, 2)
    _check_matmul(table, scales, *O.codes(x), bias, torch.float32, x.cuda())


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("tokens,rows,dim", [(300, 20_001, 64), (1100, 9001, 80), (700, 30_001, 128), (64, 40_000, 72), (2000, 1001, 48),
                                             (257, 33_000, 200)])
def test_int8_matmul_tiles(tokens, rows, dim, out):
    """Tiles of every size, in one round over the chip and in several, the last one in part."""
    H.note(f"[tower] int8_matmul {tokens} x {dim} x {rows} {out}")
    table, scales, bias = _table(rows, dim, 1)
    _check_matmul(table, scales, *O.codes(_data((tokens, dim), torch.float32, 2)), bias, out)


@pytest.mark.parametrize("tokens", [1, 20, 100])
def test_int8_matmul_extremes(tokens):
    """The longest rows with every code -128: sums of 2^31 - 2^18; mixed ones; no reads past a table's end."""
    H.note(f"[tower] int8_matmul extremes {tokens}")
    columns = (1 << 17) - 16
    table = torch.full((33, columns), -128, dtype=torch.int8)
    table[1] = 127
    table[2, ::2] = 127
    x = torch.full((tokens, columns), -128, dtype=torch.int8)
    _check_matmul(table, torch.ones(33), x, torch.full((tokens,), 2.0 ** -20), None, None)


def test_int8_matmul_values():
    """Vectors and rows whose scale is NaN, infinite or zero leave the others alone; scales far from 1; -0 and zero rows."""
    H.note("[tower] int8_matmul values")
    table, scales, bias = _table(70, 96, 1)
    scales[3], scales[4], scales[5] = math.nan, 0.0, 2.0 ** 60
    x = _data((20, 96), torch.float32, 2)
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    x[3] = 0.0
    x[4] *= 2.0 ** -100
    x[5] *= 2.0 ** 60
    codes, x_scales = O.codes(x)
    for m in (x, x[:6]):
        got = _check_matmul(table, scales, codes[:len(m)], x_scales[:len(m)], None, None, m.cuda())
        assert torch.isnan(got[1]).all() and torch.isnan(got[:, 3]).all() and not got[3, :3].any()


def test_int8_matmul_forms():
    """Vectors and batches of any shape and stride, tables of any alignment, no rows, no vectors, CPU tensors."""
    H.note("[tower] int8_matmul forms")
    table, scales, bias = _table(90, 80, 1)
    x = _data((3, 4, 80), torch.float32, 2)
    flat = x.view(12, 80)
    want = _check_matmul(table, scales, *O.codes(flat), bias, None, flat.cuda())
    t, s, b = table.cuda(), scales.cuda(), bias.cuda()
    assert torch.equal(st.int8_matmul(t, s, x.cuda(), None, b), want.view(3, 4, 90))
    assert torch.equal(st.int8_matmul(t, s, flat[5].cuda(), None, b), want[5])
    codes, x_scales = st.int8_quantize(x.cuda())
    assert torch.equal(st.int8_matmul(t, s, codes, x_scales, b), want.view(3, 4, 90))
    assert torch.equal(st.int8_matmul(t, s, *st.int8_quantize(flat[5].cuda()), b), want[5])
    assert torch.equal(st.int8_matmul(table, scales, x, None, bias), want.view(3, 4, 90).cpu())
    wide = torch.nn.functional.pad(flat, (1, 2), value=1e9).cuda()[:, 1:-2]
    assert torch.equal(st.int8_matmul(t, s, wide, None, b), want)
    moved = torch.cat([torch.zeros(5, dtype=torch.int8, device="cuda"), t.flatten()])[5:].view(90, 80)
    assert moved.data_ptr() % 16 and torch.equal(st.int8_matmul(moved, s, flat.cuda(), None, b), want)
    assert torch.equal(st.int8_matmul(t.t().contiguous().t(), s, flat.cuda(), None, b), want)
    assert torch.equal(st.int8_matmul(t, torch.stack([s, s], 1)[:, 0], flat.cuda(), None, b), want)
    odd = torch.cat([torch.zeros(7, dtype=torch.int8, device="cuda"), codes.flatten()])[7:].view(codes.shape)
    assert torch.equal(st.int8_matmul(t, s, odd, x_scales, b), want.view(3, 4, 90))
    assert st.int8_matmul(t[:0], s[:0], flat.cuda()).shape == (12, 0)
    assert st.int8_matmul(t, s, flat[:0].cuda()).shape == (0, 90)


def test_eight_bit_operators_refuse_gradients():
    H.note("[tower] int8 gradients")
    table, scales, bias = (t.cuda() for t in _table(20, 64, 1))
    x = _data((3, 64), torch.float32, 2).cuda()
    want = st.int8_matmul(table, scales, x, None, bias)
    for values in ((scales, x, bias), (scales, x.clone().requires_grad_(), bias), (scales.clone().requires_grad_(), x, bias),
                   (scales, x, bias.clone().requires_grad_())):
        y = st.int8_matmul(table, values[0], values[1], None, values[2])
        assert torch.equal(y.detach(), want)
        if y.requires_grad:
            with pytest.raises(RuntimeError, match="int8_matmul has no gradient"):
                y.sum().backward()
    leaf = x.clone().requires_grad_()
    for op, made in (("int8_quantize", st.int8_quantize(leaf)), ("layer_norm_int8", st.layer_norm_int8(leaf))):
        assert not made[0].requires_grad
        with pytest.raises(RuntimeError, match=f"{op} has no gradient"):
            made[1].sum().backward()


def test_second_derivatives_are_refused():
    H.note("[tower] second derivatives")
    x, w, s = _data((3, 40), torch.float32, 1).cuda().requires_grad_(), torch.ones(40, device="cuda", requires_grad=True), _state(1).cuda()
    for op, y in (("layer_norm", st.layer_norm(x, w)), ("dropout", st.dropout(x, 0.5, s)),
                  ("dropout_add_layer_norm", st.dropout_add_layer_norm(x, x, w, None, 0.5, s)[0])):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match=f"gradient of {op} cannot be differentiated again"):
            g.sum().backward()


# ------------------------------------------------------------------ streams and graphs


def test_streams_and_graphs():
    """A training and a serving pass on another stream, and captured: replays with new inputs and states, eager work
    between them, give the eager bits; two graphs share nothing."""
    H.note("[tower] graphs")
    rows, dim, wide = 300, 640, 1000
    w, b = _data((dim,), torch.float32, 3, 0.2, 1.0).cuda().requires_grad_(), _data((dim,), torch.float32, 4).cuda().requires_grad_()
    table, scales, bias = (t.cuda() for t in _table(wide, dim, 1))

    def step(x, res, state, gy, gs):
        y, total = st.dropout_add_layer_norm(x, res, w, b, 0.2, state)
        z = st.dropout(y, 0.3, state)
        grads = torch.autograd.grad([z, total], [x, res, w, b], [gy, gs])
        state[1] += 1
        codes, s = st.layer_norm_int8(x, w.detach(), b.detach())
        few = st.int8_matmul(table, scales, x.detach()[:3], None, bias)
        many = st.int8_matmul(table, scales, codes, s, bias, torch.bfloat16)
        made = st.int8_matmul(table, scales, x.detach(), None, None)
        return [t.detach() for t in (z, total, *grads, codes, s, few, many, made)]

    def inputs(seed):
        return [_data((rows, dim), torch.bfloat16, seed).cuda(), _data((rows, dim), torch.float32, seed + 1).cuda(),
                _state(seed).cuda(), _data((rows, dim), torch.bfloat16, seed + 2).cuda(), _data((rows, dim), torch.float32, seed + 3).cuda()]

    def eager(seed):
        x, res, state, gy, gs = inputs(seed)
        return [t.clone() for t in step(x.requires_grad_(), res.requires_grad_(), state, gy, gs)] + [state]

    side = torch.cuda.Stream()
    graphs = []
    for k in range(2):
        held = inputs(50 + k)
        leaves = [held[0].requires_grad_(), held[1].requires_grad_(), *held[2:]]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(*leaves)
            want = eager(90 + k)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(want, eager(90 + k)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*leaves)
        graphs.append((graph, held, out))
    for turn in range(4):
        for k, (graph, held, out) in enumerate(graphs):
            seed = 10 * turn + k
            fresh = inputs(seed)
            with torch.no_grad():
                for t, f in zip(held, fresh):
                    t.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            want = eager(seed)
            got = [*out, held[2]]
            for i, (p, q) in enumerate(zip(got, want)):
                assert torch.equal(p, q), (turn, k, i)
