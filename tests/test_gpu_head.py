"""The retrieval head's operators on the GPU against plain 64-bit forms
(tests/head_oracle.py): 4-bit tables, log-probabilities of given documents,
cluster routing; their gradients against autograd in 64 bits and against
differences.

Tolerances (u = 2^-24, the rounding of 32 bits):
- a log-probability, entropy or lse is a sum of terms of size R = |max z| / T +
  log columns (and of its own size), each rounded a few times, and of a sum of positive terms whose
  relative error stays below ~32 u (partial sums of at most a few hundred
  terms per thread, then a tree): 64 u (1 + R).
- a gradient's element is e^(z/T - l) (1 + relative 64 u (1 + R)) times
  coefficients that are sums of a few terms: 128 u (1 + R) times the sum of the
  absolute values of its terms, then one rounding to its type (half a unit:
  relative 2^-8 for bfloat16, 2^-11 for float16 and 2^-25 below its normal range).
- a 4-bit product of D columns: terms |q x s| with a relative error of 2^-22
  from x's parts, summed in 32 bits: (2^-22 + D u) sum |terms| bounds it, then
  one rounding to its type.
"""

import math

import pytest
import torch

from tests import gpu_helpers as H
from tests import head_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _near(got, want, atol, what=""):
    """got within atol (a number or a tensor) of want; values that are not finite, or past got's type, are the same."""
    want = want.detach().double()
    want = torch.where(want.abs() > torch.finfo(got.dtype).max, want.sign() * math.inf, want)
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), what
    atol = torch.as_tensor(atol, dtype=torch.float64).expand(want.shape)
    off = (got - want).abs()
    bad = fine & ~(off <= atol)
    assert not bad.any(), (what, off[bad][:5], atol[bad][:5], want[bad][:5])


# ------------------------------------------------------------------ log-probabilities


def _range(logits, temperature, mask=None):
    """R of each row: of its largest score that passes (smaller ones matter by their distance from it, and those
    more than ~100 T below it do not)."""
    z = logits.double()
    if mask is not None:
        z = torch.where(O.bits(mask.expand(len(z), -1), z.shape[1]), z, -math.inf)
    top = z.amax(1) if z.shape[1] else torch.zeros(len(z))
    return torch.where(torch.isfinite(top), top, 0.0).abs() / temperature + math.log(max(2, logits.shape[1]))


def _check_logprobs(logits, targets, topk, mask, temperature, grads=True, gpu_logits=None):
    """Every output and, with `grads`, the gradient of all four."""
    rows, columns = logits.shape
    x = (logits.cuda() if gpu_logits is None else gpu_logits).detach().requires_grad_(grads)
    m = mask.cuda() if mask is not None else None
    out = torch.ops.st.target_logprobs(x, targets.cuda(), topk, m, temperature)
    leaf = logits.double().requires_grad_(grads)
    want = O.target_logprobs(leaf, targets, topk, mask, temperature)
    r = _range(logits, temperature, mask)
    assert torch.equal(out[3].cpu(), want[3]), "top_ids"
    for i, what in ((0, "logprobs"), (1, "entropy"), (2, "lse"), (4, "top_logprobs")):
        size = (r.unsqueeze(1) if i == 4 else r) + torch.where(torch.isfinite(want[i]), want[i].detach(), 0.0).abs()
        _near(out[i], want[i], 64 * U * (1 + size), what)
    if not grads:
        return out
    g = torch.Generator().manual_seed(rows * 31 + columns)
    cot = [torch.randn(o.shape, generator=g) for o in (out[0], out[1], out[2], out[4])]
    got, = torch.autograd.grad([out[0], out[1], out[2], out[4]], [x], [c.cuda() for c in cot])
    assert got.dtype == logits.dtype and got.shape == logits.shape
    # 64-bit gradient of the finite outputs
    pairs = [(w, c) for w, c in zip((want[0], want[1], want[2], want[4]), cot)]
    total = sum((torch.where(torch.isfinite(w), w, 0.0) * c).sum() for w, c in pairs)
    grad = torch.autograd.grad(total, leaf)[0] if total.requires_grad else torch.zeros_like(leaf)
    # the size of each element's terms
    with torch.no_grad():
        allowed = logits != -math.inf
        if mask is not None:
            allowed &= O.bits(mask.expand(rows, -1), columns)
        z = torch.where(allowed, logits.double() / temperature, -math.inf)
        lse = torch.where(torch.isfinite(want[2]), want[2], 0.0).unsqueeze(1)
        p = torch.where(allowed, (z - lse).exp(), 0.0)
        logp = torch.where(p > 0, z - lse, 0.0)
        whole = cot[0].abs() + cot[2].abs() + cot[3].abs().sum(1)
        terms = p * (whole.unsqueeze(1) + cot[1].abs().unsqueeze(1) * (logp.abs() + want[1].unsqueeze(1)))
        at = targets.clamp(0, max(columns - 1, 0)).unsqueeze(1)
        if columns:
            terms.scatter_add_(1, at, cot[0].abs().double().unsqueeze(1))
            terms.scatter_add_(1, want[3].clamp(min=0), cot[3].abs().double())
        atol = terms / temperature * (128 * U * (1 + r.unsqueeze(1)) + HALF[logits.dtype] * 1.01) + TINY[logits.dtype]
    _near(got, grad, atol, "grad_logits")
    # excluded columns: exactly nothing
    assert not got.detach().cpu()[~allowed].any()
    return out


def _case(rows, columns, dtype, seed, scale=2.0, density=0.4):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((rows, columns), generator=g) * scale).to(dtype)
    passes = torch.rand((rows, columns), generator=g) < density
    targets = torch.randint(0, columns, (rows,), generator=g)
    passes[torch.arange(rows), targets] = True
    return logits, O.pack(passes), targets


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns,topk", [
    (1, 1, 1), (3, 7, 3), (2, 8, 8), (5, 9, 20), (4, 63, 5), (4, 64, 64), (3, 65, 0), (2, 1000, 128), (3, 2049, 33),
    (2, 8191, 7), (2, 8193, 10), (1, 50_001, 100), (1, 300_007, 32),
])
@pytest.mark.parametrize("filtered", [False, True])
def test_logprobs_and_gradient(rows, columns, topk, dtype, filtered):
    H.note(f"[logprobs] {rows} x {columns} top {topk} {dtype} filtered={filtered}")
    logits, mask, targets = _case(rows, columns, dtype, rows + columns)
    _check_logprobs(logits, targets, topk, mask if filtered else None, 0.7)


@pytest.mark.parametrize("rows,columns", [(2100, 130), (2050, 1001), (300, 3000), (600, 20_000)])
def test_logprobs_many_rows(rows, columns):
    """Rows enough for the kernels' other grids."""
    H.note(f"[logprobs] {rows} x {columns}")
    logits, mask, targets = _case(rows, columns, torch.bfloat16, 5)
    _check_logprobs(logits, targets, 9, mask, 1.0)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 30.0])
def test_logprobs_temperature(temperature):
    H.note(f"[logprobs] temperature {temperature}")
    logits, mask, targets = _case(4, 3000, torch.float32, 8)
    _check_logprobs(logits, targets, 12, mask, temperature)


@pytest.mark.parametrize("columns", [40, 5000, 70_000])
@pytest.mark.parametrize("topk", [1, 40, 128])
def test_logprobs_equal_scores(columns, topk):
    """All scores equal, or of two values: alternatives are the lowest columns."""
    H.note(f"[logprobs] ties {columns} top {topk}")
    for logits in (torch.zeros((2, columns)), torch.randint(0, 2, (2, columns), generator=torch.Generator().manual_seed(3)).float()):
        _check_logprobs(logits, torch.tensor([0, columns - 1]), topk, None, 1.0)
    # -0 and +0 are equal
    logits = torch.zeros((1, columns))
    logits[0, ::2] = -0.0
    _check_logprobs(logits, torch.tensor([1]), topk, None, 1.0)


@pytest.mark.parametrize("order", ["up", "down", "strided"])
@pytest.mark.parametrize("rows,columns", [(1, 40_000), (2100, 2500)])
def test_logprobs_orders(order, rows, columns):
    """Scores sorted either way, and all the large ones in few threads' columns."""
    H.note(f"[logprobs] order {order} {rows} x {columns}")
    z = torch.arange(columns, dtype=torch.float32) / columns * 8
    if order == "down":
        z = z.flip(0)
    if order == "strided":
        at = torch.arange(columns)
        z = torch.where(at // 8 % 256 < 40, 5 + z / 8, z / 8)
    _check_logprobs(z.repeat(rows, 1), torch.full((rows,), 17), 100, None, 1.0, grads=rows == 1)


@pytest.mark.parametrize("rows,columns,threads", [(1, 65_536, 1024), (2100, 20_001, 256)])
def test_logprobs_high_scores_in_few_threads(rows, columns, threads):
    """Every score of 40 threads' columns above all others, and more alternatives wanted than that: the candidates
    outgrow their list."""
    H.note(f"[logprobs] few threads {rows} x {columns}")
    at = torch.arange(columns)
    noise = torch.randperm(columns, generator=torch.Generator().manual_seed(5)).float() / columns
    z = torch.where(at // 8 % threads < 40, 10 + noise, noise)
    _check_logprobs(z.repeat(rows, 1), torch.full((rows,), 17), 100, None, 1.0, grads=rows == 1)


def test_logprobs_excluded_places():
    """Rows that nothing passes, infinities and NaN behind the filter, the type's lowest value, -inf among what
    passes, targets that are masked, -inf, out of range and absent."""
    H.note("[logprobs] excluded places")
    rows, columns = 12, 700
    logits, mask, targets = _case(rows, columns, torch.float32, 21)
    passes = O.bits(mask, columns)
    logits = torch.where(passes, logits, torch.tensor([math.nan, math.inf, -math.inf, 3e38]).repeat(rows, columns // 4))
    passes[0] = False                                   # nothing passes
    passes[1] = False
    passes[1, 699] = True                               # one document
    logits[2] = torch.where(passes[2], -math.inf, logits[2])   # all that pass at -inf
    logits[3, :350] = -math.inf
    logits[4] = torch.finfo(torch.float32).min          # the lowest value everywhere
    logits[5, ::2] = torch.where(passes[5, ::2], torch.finfo(torch.float32).min, logits[5, ::2])
    logits[6, int(targets[6])] = -math.inf
    masked = (~passes[7]).nonzero().flatten()[0]
    targets = targets.clone()
    targets[7], targets[8], targets[9], targets[10], targets[11] = masked, -1, columns, -2, 1 << 40
    targets[1] = 699
    for topk in (0, 3, 100):
        out = _check_logprobs(logits, targets, topk, O.pack(passes), 0.9)
        assert out[0][0].item() == -math.inf and out[1][0].item() == 0 and out[2][0].item() == -math.inf
        assert out[0][1].item() == 0.0 and out[0][8].item() == 0.0


@pytest.mark.parametrize("rows,columns", [(3, 500), (3, 50_000)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_logprobs_bad_values(rows, columns, value):
    """NaN or +inf among what passes: that row says NaN, the others nothing of it; NaN is no alternative."""
    H.note(f"[logprobs] {value} {rows} x {columns}")
    logits, mask, targets = _case(rows, columns, torch.float32, 4)
    logits[1, int(targets[1])] = value
    got = torch.ops.st.target_logprobs(logits.cuda().requires_grad_(), targets.cuda(), 6, mask.cuda(), 1.0)
    for o in (got[0], got[1], got[2]):
        assert torch.isnan(o[1]) and not torch.isnan(o[0]) and not torch.isnan(o[2])
    want = O.best(torch.where(O.bits(mask, columns), logits.double(), -math.inf), 6)[0]
    assert torch.equal(got[3].cpu(), want)
    assert torch.isnan(got[4][1]).all()


def test_logprobs_no_rows_or_columns():
    H.note("[logprobs] empty")
    e = torch.ops.st.target_logprobs(torch.empty((0, 5), device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"), 3)
    assert e[0].shape == (0,) and e[3].shape == (0, 3)
    x = torch.empty((2, 0), device="cuda", requires_grad=True)
    out = torch.ops.st.target_logprobs(x, torch.tensor([-1, 0], device="cuda"), 2)
    assert out[0].tolist() == [0.0, -math.inf] and out[1].tolist() == [0, 0] and out[3].tolist() == [[-1, -1]] * 2
    assert torch.autograd.grad(out[0].sum(), x)[0].shape == (2, 0)


def test_logprobs_strides_and_shared_mask():
    """Rows of a wider tensor at an odd offset, transposed scores, one mask row for all, strided mask rows,
    gradients of a broadcast input."""
    H.note("[logprobs] strides")
    logits, mask, targets = _case(6, 1001, torch.bfloat16, 77)
    wide = torch.full((6, 1205), math.nan, dtype=torch.bfloat16)
    wide[:, 3:1004] = logits
    _check_logprobs(logits, targets, 5, mask, 1.0, gpu_logits=wide.cuda()[:, 3:1004])
    _check_logprobs(logits, targets, 5, mask, 1.0, gpu_logits=logits.t().contiguous().cuda().t())
    passes = O.bits(mask, 1001)[:1]
    shared = O.pack(passes)
    _check_logprobs(logits, targets, 5, shared, 1.0)
    m = torch.zeros((6, 77), dtype=torch.int64)
    m[:, 5:5 + mask.shape[1]] = mask
    x = logits.cuda()
    a = torch.ops.st.target_logprobs(x, targets.cuda(), 5, m.cuda()[:, 5:5 + mask.shape[1]], 1.0)
    b = torch.ops.st.target_logprobs(x, targets.cuda(), 5, mask.cuda(), 1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    row = logits[:1].float()
    leaf = row.cuda().requires_grad_()
    out = torch.ops.st.target_logprobs(leaf.expand(6, -1), targets.cuda(), 5, mask.cuda(), 1.0)
    got, = torch.autograd.grad(out[0].sum(), leaf)
    ref = row.double().requires_grad_()
    want = O.target_logprobs(ref.expand(6, -1), targets, 5, mask, 1.0)
    grad, = torch.autograd.grad(torch.where(torch.isfinite(want[0]), want[0], 0.0).sum(), ref)
    _near(got, grad, 6 * 128 * U * 20, "broadcast gradient")


def test_logprobs_offsets_past_32_bits():
    """The last rows of scores whose element offsets pass 2^31."""
    H.note("[logprobs] offsets past 2^31")
    rows, columns = 2200, 1_000_003
    x = torch.zeros((rows, columns), dtype=torch.bfloat16, device="cuda")
    tail, _, _ = _case(2, columns, torch.bfloat16, 2)
    x[-2:] = tail.cuda()
    targets = torch.full((rows,), columns - 1, device="cuda")
    x.requires_grad_()
    out = torch.ops.st.target_logprobs(x, targets, 4)
    want = O.target_logprobs(tail.double(), torch.full((2,), columns - 1), 4)
    r = 30.0
    assert torch.equal(out[3][-2:].cpu(), want[3])
    for i in (0, 1, 2, 4):
        _near(out[i][-2:], want[i], 64 * U * (1 + r))
    _near(out[2][:1], torch.tensor([math.log(columns)]), 64 * U * (1 + r))
    got, = torch.autograd.grad(out[0].sum(), x)
    p = torch.softmax(tail.double(), 1)
    p[:, -1] -= 1
    _near(got[-2:], -p, p.abs() * (HALF[torch.bfloat16] * 1.01 + 128 * U * (1 + r)) + 1e-37)


def test_logprobs_gradient_against_differences():
    """The directional derivative: central differences of the operator itself.  With step h along a direction of
    unit elements' scale, the third derivative's share is h^2 / 6 times at most a few, and each output's rounding
    64 u (1 + R) over h."""
    H.note("[logprobs] differences")
    logits, mask, targets = _case(4, 257, torch.float32, 9, scale=1.0)
    g = torch.Generator().manual_seed(1)
    way = torch.randn(logits.shape, generator=g)
    way /= way.abs().max()
    cot = [torch.rand(4, generator=g), torch.rand(4, generator=g), torch.rand(4, generator=g), torch.rand((4, 6), generator=g)]
    ids = torch.ops.st.target_logprobs(logits.cuda(), targets.cuda(), 6, mask.cuda(), 0.8)[3]

    def value(z):
        o = torch.ops.st.target_logprobs(z.cuda(), targets.cuda(), 6, mask.cuda(), 0.8)
        # the alternatives of the middle point, read from their own calls
        tops = torch.stack([torch.ops.st.target_logprobs(z.cuda(), ids[:, i].contiguous(), 0, mask.cuda(), 0.8)[0]
                            for i in range(6)], 1)
        return sum((a.cpu().double() * c.double()).sum().item() for a, c in zip((o[0], o[1], o[2], tops), cot))

    x = logits.cuda().requires_grad_()
    o = torch.ops.st.target_logprobs(x, targets.cuda(), 6, mask.cuda(), 0.8)
    grad, = torch.autograd.grad([o[0], o[1], o[2], o[4]], [x], [c.cuda() for c in cot])
    h = 2.0 ** -6
    slope = (value(logits + h * way) - value(logits - h * way)) / (2 * h)
    outputs = 4 * 9
    assert abs(slope - (grad.cpu().double() * way.double()).sum().item()) < outputs * (h * h + 64 * U * 12 / h)


def test_logprobs_some_gradients():
    """Outputs that no loss reads give nothing."""
    H.note("[logprobs] partial gradients")
    logits, mask, targets = _case(3, 900, torch.float32, 13)
    for which in range(5):
        if which == 3:
            continue
        x = logits.cuda().requires_grad_()
        o = torch.ops.st.target_logprobs(x, targets.cuda(), 4, mask.cuda(), 1.0)
        got, = torch.autograd.grad(o[which].sum(), x)
        leaf = logits.double().requires_grad_()
        w = O.target_logprobs(leaf, targets, 4, mask, 1.0)
        grad, = torch.autograd.grad(w[which].sum(), leaf)
        _near(got, grad, 128 * U * 20 * 5, which)
    with torch.no_grad():
        assert not torch.ops.st.target_logprobs(x, targets.cuda())[0].requires_grad


# ------------------------------------------------------------------ routing


def _check_route(logits, probes, valid=None, grads=True, gpu_logits=None):
    x = (logits.cuda() if gpu_logits is None else gpu_logits).detach().requires_grad_(grads)
    out = torch.ops.st.cluster_route(x, probes, valid.cuda() if valid is not None else None)
    leaf = logits.double().requires_grad_(grads)
    want = O.cluster_route(leaf, probes, valid)
    r = _range(logits, 1.0)
    if valid is not None:
        r = torch.where(valid, r, 0.0)
    assert torch.equal(out[0].cpu(), want[0]), "ids"
    assert torch.equal(out[3].cpu(), want[3]), "counts"
    _near(out[1], want[1], 64 * U * (1 + r.unsqueeze(1)) * want[1].detach() + 1e-37, "weights")
    _near(out[2], want[2], 64 * U * (1 + r), "lse")
    # a sum over rows of rounded probabilities: relative 64 u (1 + R), and u for each addition of a workgroup's rows
    rows = max(1, logits.shape[0])
    widest = float(r.max()) if len(r) else 0.0
    _near(out[4], want[4], U * (64 * (1 + widest) + min(rows, 4096)) * want[4].detach().abs() + 1e-37, "loss")
    if not grads:
        return out
    g = torch.Generator().manual_seed(rows)
    cot = [torch.randn(out[1].shape, generator=g), torch.randn(out[2].shape, generator=g), torch.tensor(1.7)]
    got, = torch.autograd.grad([out[1], out[2], out[4]], [x], [c.cuda() for c in cot])
    total = sum((torch.where(torch.isfinite(w), w, 0.0) * c).sum() for w, c in zip((want[1], want[2], want[4]), cot))
    grad = torch.autograd.grad(total, leaf)[0] if total.requires_grad else torch.zeros_like(leaf)
    with torch.no_grad():
        on = torch.isfinite(want[2])
        p = torch.where(on.unsqueeze(1), torch.exp(logits.double() - torch.where(on, want[2], 0.0).unsqueeze(1)), 0.0)
        n = max(1, int(on.sum()))
        slope = 1.7 * logits.shape[1] * want[3].double() / (probes * n * n)
        a = slope.expand_as(p).clone()
        a.scatter_add_(1, want[0].clamp(min=0), torch.where(want[0] >= 0, cot[0].abs().double(), 0.0))
        terms = p * (a + (p * a).sum(1, keepdim=True) + cot[1].abs().unsqueeze(1))
        atol = terms * (128 * U * (1 + r.unsqueeze(1)) + HALF[logits.dtype] * 1.01) + TINY[logits.dtype]
    _near(got, grad, atol, "grad_logits")
    assert not got.cpu()[~on].any()
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,clusters,probes", [
    (1, 1, 1), (3, 5, 2), (130, 8, 8), (5, 64, 64), (257, 65, 9), (33, 128, 3), (140, 129, 17), (9, 256, 40),
    (20, 257, 5), (17, 512, 64), (33, 513, 8), (50, 1000, 1), (18, 1024, 24), (7, 1025, 33), (19, 2048, 16),
    (5, 2049, 16), (9, 4096, 31), (6, 4097, 64), (5, 8192, 12), (3, 8193, 20), (2, 16_384, 64), (3, 16_385, 7),
    (2, 32_768, 50),
])
def test_route_and_gradient(rows, clusters, probes, dtype):
    H.note(f"[route] {rows} x {clusters} probes {probes} {dtype}")
    g = torch.Generator().manual_seed(rows + clusters)
    logits = (torch.randn((rows, clusters), generator=g) * 2).to(dtype)
    _check_route(logits, probes)
    _check_route(logits, probes, torch.rand(rows, generator=g) < 0.6)


@pytest.mark.parametrize("rows,clusters,probes", [(9000, 60, 4), (5000, 300, 5), (3000, 2500, 8)])
def test_route_many_rows(rows, clusters, probes):
    H.note(f"[route] {rows} x {clusters}")
    logits = torch.randn((rows, clusters), generator=torch.Generator().manual_seed(4)) * 3
    _check_route(logits, probes, torch.arange(rows) % 7 != 3)


@pytest.mark.parametrize("clusters", [8, 100, 700, 3000, 20_000])
@pytest.mark.parametrize("probes", [1, 8, 64])
def test_route_equal_scores(clusters, probes):
    """All scores equal, or of two values: the lowest clusters."""
    H.note(f"[route] ties {clusters} probes {probes}")
    _check_route(torch.zeros((5, clusters)), probes)
    _check_route(torch.randint(0, 2, (5, clusters), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16), probes)


@pytest.mark.parametrize("clusters,probes,lanes,period", [(1024, 8, 5, 16), (2048, 30, 20, 64), (5000, 24, 80, 256),
                                                          (30_000, 40, 300, 1024)])
def test_route_high_scores_in_few_lanes(clusters, probes, lanes, period):
    """Every score of a few lanes' clusters above all others, so that far more than the probes reach the bound."""
    H.note(f"[route] few lanes {clusters} probes {probes}")
    at = torch.arange(clusters)
    g = torch.Generator().manual_seed(7)
    noise = torch.stack([torch.randperm(clusters, generator=g) for _ in range(9)]).float() / clusters
    _check_route(torch.where(at // 8 % period < lanes, 3 + noise, noise), probes, torch.arange(9) != 4)


@pytest.mark.parametrize("clusters", [40, 600, 5000])
def test_route_excluded(clusters):
    """Clusters at -inf are not chosen, rows with fewer left are padded, rows without any are not counted; flags off
    hide NaN; the lowest value is a score like any other."""
    H.note(f"[route] excluded {clusters}")
    logits = torch.randn((8, clusters), generator=torch.Generator().manual_seed(6))
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, ::2] = -math.inf
    logits[3] = torch.finfo(torch.float32).min
    logits[4, :-1] = torch.finfo(torch.float32).min
    valid = torch.ones(8, dtype=torch.bool)
    valid[5] = False
    hidden = logits.clone()
    out = _check_route(logits, 12, valid)
    hidden[5] = math.nan
    again = torch.ops.st.cluster_route(hidden.cuda(), 12, valid.cuda())
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    none = torch.ops.st.cluster_route(logits.cuda(), 12, torch.zeros(8, dtype=torch.bool, device="cuda"))
    assert (none[0] == -1).all() and not none[1].any() and not none[3].any() and none[4].item() == 0
    # a NaN among a row's scores: the row's and the loss's numbers say so, and it is never chosen
    logits[6, 1] = math.nan
    bad = torch.ops.st.cluster_route(logits.cuda(), 12, valid.cuda())
    assert torch.isnan(bad[2][6]) and torch.isnan(bad[4]) and not (bad[0][6] == 1).any() and torch.isfinite(bad[2][7])


def test_route_no_rows():
    H.note("[route] no rows")
    x = torch.empty((0, 9), device="cuda", requires_grad=True)
    out = torch.ops.st.cluster_route(x, 2)
    assert out[0].shape == (0, 2) and out[3].tolist() == [0] * 9 and out[4].item() == 0
    assert torch.autograd.grad(out[4], x)[0].shape == (0, 9)


def test_route_strides_and_repeats():
    """Odd rows of a wider tensor; the same inputs give the same bits."""
    H.note("[route] strides")
    logits = torch.randn((40, 1001), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    wide = torch.full((40, 1101), math.nan, dtype=torch.bfloat16)
    wide[:, 7:1008] = logits
    _check_route(logits, 9, gpu_logits=wide.cuda()[:, 7:1008])
    _check_route(logits, 9, gpu_logits=logits.t().contiguous().cuda().t())
    big = torch.randn((4000, 777), generator=torch.Generator().manual_seed(2)).cuda()
    a, b = (torch.ops.st.cluster_route(big, 5) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_route_gradient_against_differences():
    """With the counts constant, as they are where no choice changes: a step that leaves the ids alone."""
    H.note("[route] differences")
    g = torch.Generator().manual_seed(12)
    logits = torch.stack([torch.randperm(40, generator=g) for _ in range(6)]).float() * 0.25
    way = torch.rand((6, 40), generator=g) * 2 - 1
    cot = [torch.rand((6, 3), generator=g), torch.rand(6, generator=g), torch.tensor(2.0)]

    def outputs(z):
        o = torch.ops.st.cluster_route(z, 3)
        return o[0], [o[1], o[2], o[4]]

    x = logits.cuda().requires_grad_()
    ids, o = outputs(x)
    grad, = torch.autograd.grad(o, [x], [c.cuda() for c in cot])
    h = 2.0 ** -5
    ends = []
    for sign in (1, -1):
        i, e = outputs((logits + sign * h * way).cuda())
        assert torch.equal(i, ids)
        ends.append(sum((a.cpu().double() * c.double()).sum().item() for a, c in zip(e, cot)))
    slope = (ends[0] - ends[1]) / (2 * h)
    assert abs(slope - (grad.cpu().double() * way.double()).sum().item()) < 25 * (h * h + 64 * U * 15 / h)


def test_second_derivatives_refused():
    """A graph over the gradients is allowed; going back through it says that it cannot be."""
    H.note("[head] second derivatives")
    for device in ("cuda", "cpu"):
        x = torch.randn((3, 50), generator=torch.Generator().manual_seed(1)).to(device).requires_grad_()
        targets = torch.arange(3, device=device)
        for name, output in (("target_logprobs", lambda: torch.ops.st.target_logprobs(x, targets)[0]),
                             ("cluster_route", lambda: torch.ops.st.cluster_route(x, 4)[2])):
            plain, = torch.autograd.grad(output().sum(), x)
            once, = torch.autograd.grad(output().sum(), x, create_graph=True)
            assert torch.equal(plain, once) and not plain.requires_grad
            with pytest.raises(RuntimeError, match=f"gradient of {name} cannot be differentiated again"):
                torch.autograd.grad(once.square().sum(), x)


# ------------------------------------------------------------------ 4-bit tables


def _table(n, dim, group, scale_type, asymmetric, seed):
    g = torch.Generator().manual_seed(seed)
    groups = -(-dim // group)
    packed = torch.randint(0, 256, (n, -(-dim // 32) * 16), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, groups), generator=g) + 0.5).to(scale_type)
    zeros = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if asymmetric else None
    return packed, scales, zeros


def _check_matvec(packed, scales, zeros, x, group, out_type=None):
    dim = x.shape[-1]
    y = torch.ops.st.int4_matvec(packed.cuda(), scales.cuda(), x.cuda(), group,
                                 zeros.cuda() if zeros is not None else None, out_type)
    w = O.dequantize(packed, scales, zeros, dim, group)
    want = x.double() @ w.T.contiguous()
    size = x.double().abs() @ w.abs().T.contiguous()
    t = out_type or x.dtype
    assert y.dtype == t
    _near(y, want, size * (2.0 ** -22 + dim * U) + want.abs() * HALF[t] * 1.01 + TINY[t], (packed.shape, x.shape))
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("asymmetric", [False, True])
@pytest.mark.parametrize("n,dim,group,queries", [
    (1, 1, 32, 1), (3, 31, 32, 1), (17, 32, 64, 2), (100, 33, 32, 3), (65, 64, 64, 16), (1000, 100, 32, 5),
    (513, 128, 128, 1), (2047, 128, 32, 17), (300, 256, 96, 33), (129, 777, 256, 4), (1030, 1024, 128, 1),
    (77, 4096, 32, 9), (50, 8200, 64, 64), (40, 8192, 8192, 1), (5, 20_001, 128, 2), (1, 300, 32, 70),
])
def test_matvec(n, dim, group, queries, asymmetric, dtype):
    H.note(f"[int4] {n} x {dim} group {group} queries {queries} zeros={asymmetric} {dtype}")
    packed, scales, zeros = _table(n, dim, group, dtype, asymmetric, n + dim)
    x = torch.randn((queries, dim), generator=torch.Generator().manual_seed(dim)).to(dtype)
    _check_matvec(packed, scales, zeros, x, group)
    _check_matvec(packed, scales, zeros, x, group, torch.float32)
    _check_matvec(packed, scales, zeros, x[0], group)


@pytest.mark.parametrize("n,dim,queries,dtype", [
    (1000, 1024, 64, torch.bfloat16), (1000, 900, 63, torch.float16), (1000, 1000, 32, torch.float32),
    (33_000, 1024, 64, torch.bfloat16), (500, 1536, 42, torch.bfloat16), (500, 2048, 32, torch.float16),
    (200, 4096, 16, torch.bfloat16), (200, 4097, 8, torch.float32),
])
def test_matvec_vectors_that_fill_lds(n, dim, queries, dtype):
    """As many vectors as are held at once, beside the sums of the waves that share rows."""
    H.note(f"[int4] full LDS {n} x {dim} queries {queries} {dtype}")
    packed, scales, zeros = _table(n, dim, 64, torch.bfloat16, True, n + dim)
    x = torch.randn((queries, dim), generator=torch.Generator().manual_seed(dim)).to(dtype)
    _check_matvec(packed, scales, zeros, x, 64, torch.float32)


@pytest.mark.parametrize("n,dim,queries,dtype", [
    (500, 2100, 64, torch.bfloat16), (3000, 1100, 65, torch.float16), (9000, 2100, 33, torch.bfloat16),
    (700, 2100, 33, torch.float32), (17_000, 1100, 64, torch.bfloat16),
])
def test_matvec_many_long_vectors(n, dim, queries, dtype):
    """Vectors that LDS cannot hold at once, taken in passes or in phases."""
    H.note(f"[int4] long vectors {n} x {dim} queries {queries} {dtype}")
    packed, scales, zeros = _table(n, dim, 64, torch.bfloat16, True, n + dim)
    x = torch.randn((queries, dim), generator=torch.Generator().manual_seed(dim)).to(dtype)
    _check_matvec(packed, scales, zeros, x, 64, torch.float32)


@pytest.mark.parametrize("n", [1, 15, 16, 63, 4096, 70_001, 600_000])
@pytest.mark.parametrize("dim,queries", [(64, 1), (128, 7), (128, 16)])
def test_matvec_row_counts(n, dim, queries):
    H.note(f"[int4] rows {n} x {dim} queries {queries}")
    packed, scales, zeros = _table(n, dim, 32, torch.float16, True, n)
    x = torch.randn((queries, dim), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16)
    _check_matvec(packed, scales, zeros, x, 32, torch.float32)


@pytest.mark.parametrize("x_type,scale_type,out_type", [
    (torch.bfloat16, torch.float32, torch.float16), (torch.float16, torch.bfloat16, torch.bfloat16),
    (torch.float32, torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16, torch.float32)])
def test_matvec_types(x_type, scale_type, out_type):
    H.note(f"[int4] types {x_type} {scale_type} {out_type}")
    packed, scales, zeros = _table(200, 160, 64, scale_type, True, 1)
    x = torch.randn((3, 160), generator=torch.Generator().manual_seed(0)).to(x_type) * 0.01
    _check_matvec(packed, scales, zeros, x, 64, out_type)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matvec_ranges(dtype):
    """Vectors whose elements span the type's range: the sum's error stays relative to its largest terms."""
    H.note(f"[int4] ranges {dtype}")
    packed, scales, _ = _table(120, 256, 32, torch.float32, False, 3)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((4, 256), generator=g) * torch.exp2(torch.randint(-60, 60, (4, 256), generator=g).float())
    for x in (wide, wide * 2.0 ** 60, wide * 2.0 ** -60, torch.randn((4, 256), generator=g) * 2.0 ** -140,
              torch.zeros((4, 256))):
        _check_matvec(packed, scales, None, x.to(dtype), 32, torch.float32)
    x = torch.zeros((2, 256))
    x[0, 17] = 1e-30
    x[1, 200] = 3e38
    _check_matvec(packed, scales * 0.01, None, x.to(dtype), 32, torch.float32)


def test_matvec_bad_values():
    """NaN and infinities in a vector reach its own products only; a NaN scale its own row."""
    H.note("[int4] bad values")
    packed, scales, _ = _table(64, 128, 32, torch.float32, False, 3)
    x = torch.randn((4, 128), generator=torch.Generator().manual_seed(1))
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    scales[7, 1] = math.nan
    y = torch.ops.st.int4_matvec(packed.cuda(), scales.cuda(), x.cuda(), 32).cpu()
    want = x.double() @ O.dequantize(packed, scales, None, 128, 32).T.contiguous()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isinf(y), torch.isinf(want)) and torch.equal(y[torch.isinf(y)].double(), want[torch.isinf(want)])
    rest = torch.isfinite(want)
    assert (y[rest] - want[rest]).abs().max() < 1e-2


def test_matvec_layouts():
    """Strided scales and vectors, a table at an odd address, no rows, no vectors."""
    H.note("[int4] layouts")
    packed, scales, zeros = _table(90, 96, 32, torch.bfloat16, True, 8)
    x = torch.randn((6, 96), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    want = torch.ops.st.int4_matvec(packed.cuda(), scales.cuda(), x.cuda(), 32, zeros.cuda())
    buf = torch.zeros(packed.numel() + 16, dtype=torch.uint8, device="cuda")
    odd = buf[3:3 + packed.numel()].view_as(packed)
    odd.copy_(packed)
    got = torch.ops.st.int4_matvec(odd, scales.t().contiguous().cuda().t(), x.t().contiguous().cuda().t(), 32,
                                   zeros.t().contiguous().cuda().t())
    assert torch.equal(got, want)
    xo = torch.zeros(6 * 96 + 1, dtype=torch.bfloat16, device="cuda")
    xo[1:] = x.flatten().cuda()
    assert torch.equal(torch.ops.st.int4_matvec(packed.cuda(), scales.cuda(), xo[1:].view(6, 96), 32, zeros.cuda()), want)
    assert torch.ops.st.int4_matvec(packed[:0].cuda(), scales[:0].cuda(), x.cuda(), 32).shape == (6, 0)
    assert torch.ops.st.int4_matvec(packed.cuda(), scales.cuda(), x[:0].cuda(), 32).shape == (0, 90)


def test_matvec_offsets_past_32_bits():
    """A table of more than 2^31 bytes, and outputs past 2^31 bytes."""
    H.note("[int4] offsets past 2^31")
    n, dim = 34_000_001, 128
    packed = torch.zeros((n, 64), dtype=torch.uint8, device="cuda")
    scales = torch.ones((n, 1), dtype=torch.bfloat16, device="cuda")
    tail, ts, _ = _table(5, dim, 128, torch.bfloat16, False, 6)
    packed[-5:], scales[-5:] = tail.cuda(), ts.cuda()
    x = torch.randn((17, dim), generator=torch.Generator().manual_seed(2))
    y = torch.ops.st.int4_matvec(packed, scales, x.cuda(), 128)
    want = x.double() @ O.dequantize(tail, ts, None, dim, 128).T.contiguous()
    size = x.double().abs() @ O.dequantize(tail, ts, None, dim, 128).abs().T.contiguous()
    _near(y[:, -5:], want, size * (2.0 ** -22 + dim * U))
    rest = -8 * x.double().sum(1, keepdim=True).expand(-1, 3)
    _near(y[:, :3], rest, 8 * x.double().abs().sum(1, keepdim=True) * (2.0 ** -22 + dim * U))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("n,dim,group", [(1, 1, 32), (5, 31, 32), (40, 100, 64), (33, 256, 32), (9, 1000, 128)])
def test_quantize(n, dim, group, symmetric, dtype):
    """Bit for bit the rule in IEEE 32-bit arithmetic, whole groups of zeros and values that are not finite among
    them; codes past the last column are 0."""
    H.note(f"[int4] quantize {n} x {dim} group {group} symmetric={symmetric} {dtype}")
    w = torch.randn((n, dim), generator=torch.Generator().manual_seed(n + dim)).to(dtype)
    if n > 3:
        w[1] = 0
        w[2, dim // 2] = math.nan
        w[3, 0] = -math.inf
        w[4] = w[4].abs()
    p, s, z = (t.cpu() for t in torch.ops.st.int4_quantize(w.cuda(), group, symmetric))
    q, ws, wz = O.quantize(w, group, symmetric)
    fine = torch.isfinite(ws.float())
    assert torch.equal(torch.isnan(s.float()), torch.isnan(ws.float())) and torch.equal(s[fine], ws[fine])
    assert torch.equal(z[fine], wz[fine])
    of = torch.arange(dim) // group
    codes = O.unpack4(p, dim)
    assert torch.equal(codes[fine[:, of]], q[fine[:, of]])
    assert not O.unpack4(p, p.shape[1] * 2)[:, dim:].any()
    if symmetric and dtype == torch.float32:
        ok = fine[:, of]
        err = (O.dequantize(p, s, z, dim, group) - w.double()).abs()
        assert (err <= s.double()[:, of] * 0.5000001)[ok].all()


# ------------------------------------------------------------------ streams, graphs, CPU tensors, the module


def test_other_stream_and_graph():
    """Calls on a side stream, and recorded into a graph that is replayed several times with eager work between."""
    H.note("[head] stream and graph")
    logits, mask, targets = _case(3, 40_000, torch.float32, 3)
    packed, scales, zeros = (t.cuda() for t in _table(3000, 128, 32, torch.float16, True, 1))
    xs = torch.randn((2, 128)).cuda()
    z, m, t = logits.cuda(), mask.cuda(), targets.cuda()
    route = torch.randn((64, 600)).cuda()

    def calls():
        return [*torch.ops.st.target_logprobs(z, t, 9, m, 0.5), torch.ops.st.int4_matvec(packed, scales, xs, 32, zeros),
                *torch.ops.st.cluster_route(route, 5)]

    want = [o.clone() for o in calls()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = calls()
    for turn in range(4):
        z.copy_((logits * (1 + turn)).cuda())
        route.copy_(torch.randn((64, 600), generator=torch.Generator().manual_seed(turn)).cuda())
        eager = [o.clone() for o in calls()]
        torch.cuda.synchronize()
        for o in recorded:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, eager)), turn


def test_cpu_tensors():
    """CPU tensors give the GPU's results, gradients too."""
    H.note("[head] cpu tensors")
    logits, mask, targets = _case(3, 500, torch.float32, 3)
    outs = []
    for d in ("cpu", "cuda"):
        x = logits.to(d).requires_grad_()
        o = torch.ops.st.target_logprobs(x, targets.to(d), 4, mask.to(d), 1.0)
        r = torch.ops.st.cluster_route(x, 4)
        g, = torch.autograd.grad(o[0].sum() + o[1].sum() + r[4] + r[1].sum(), x)
        w = torch.ops.st.int4_quantize(logits.to(d), 64)
        y = torch.ops.st.int4_matvec(w[0], w[1], logits.to(d), 64, w[2])
        assert all(v.device.type == d for v in (*o, *r, g, *w, y))
        outs.append([v.cpu() for v in (*o, *r, g, *w, y)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_module():
    """A table from embeddings, saved and loaded into a new module, answering filtered queries."""
    H.note("[head] module")
    from silvertorch_amd.modules import RetrievalHeadModule

    g = torch.Generator().manual_seed(3)
    docs = torch.randn((3000, 64), generator=g)
    head = RetrievalHeadModule(group_size=32, topk=5, temperature=0.5)
    head.set_embeddings(docs.cuda())
    other = RetrievalHeadModule(group_size=32, topk=5, temperature=0.5).cuda()
    other.load_state_dict(head.state_dict())
    q = torch.randn((4, 64), generator=g).cuda()
    passes = torch.rand((4, 3000), generator=g) < 0.3
    targets = passes.float().argmax(1)
    out = other(q, targets.cuda(), O.pack(passes).cuda())
    table = O.dequantize(head.packed.cpu(), head.scales.cpu(), head.zeros.cpu(), 64, 32)
    want = O.target_logprobs(other.scores(q).cpu().double(), targets, 5, O.pack(passes), 0.5)
    assert (other.scores(q).cpu().double() - q.cpu().double() @ table.T.contiguous()).abs().max() < 1e-4
    assert torch.equal(out[3].cpu(), want[3])
    for i in (0, 1, 2, 4):
        _near(out[i], want[i], 64 * U * 100)
    assert torch.equal(other(q)[0].cpu(), torch.zeros(4))


def test_example():
    """Training lowers the loss; answers pass the filter and give the clicked document more than the uniform share."""
    H.note("[head] example")
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "retrieval_head.py"
    spec = importlib.util.spec_from_file_location("retrieval_head_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    out = module.main(["--docs", "3000", "--pairs", "256", "--steps", "40"])
    assert out["last"] < out["first"] - 1
    topics, clicked, ids = out["topics"].cpu(), out["clicked"].cpu(), out["top_ids"].cpu()
    passes = O.bits(out["mask"].cpu(), 3000)
    assert passes.gather(1, ids).all() and passes.gather(1, clicked.unsqueeze(1)).all()
    same = topics.unsqueeze(0) == topics[clicked].unsqueeze(1)
    assert (passes | ~same).all()  # a bloom filter passes every document of the topic
    assert (out["logprobs"].cpu() > -torch.log(passes.sum(1).float())).float().mean() > 0.8
