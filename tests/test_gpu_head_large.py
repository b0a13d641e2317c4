"""The retrieval head's operators at scores that are large against the temperature, or share a large offset, against
plain 64-bit forms (tests/head_oracle.py).

Probabilities and their gradients depend on the scores' distances alone, so none of the tolerances here grows with an
offset (u = 2^-24, the rounding of 32 bits; L = log columns):
- an exponential's argument d = (z - max) / T, in units of log 2, has a few roundings of relative u, which moves the
  exponential by a few u |d|; a sum of them is dominated by terms of |d| below a few L, and its additions stay below
  32 u (a few hundred terms a thread, then a tree).  A log-probability is such a sum's logarithm and one distance of its own
  size: 64 u (1 + L + |value|); the entropy is a difference of two values of size L: 64 u (1 + 2 L); lse has the offset
  itself: 64 u (1 + L + |value|).
- a probability has the relative error 64 u (1 + L + |log p|), and a gradient's element twice that of the sum of the
  absolute values of its terms, then one rounding to its type.
"""

import math

import pytest
import torch

from tests import gpu_helpers as H
from tests import head_oracle as O
from tests.test_gpu_head import HALF, TINY, TYPES, U, _near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


# ------------------------------------------------------------------ log-probabilities


def _check_logprobs(logits, targets, topk, mask, temperature):
    """Every output, and the gradient of all four."""
    rows, columns = logits.shape
    wide = math.log(max(2, columns))
    x = logits.cuda().requires_grad_()
    out = torch.ops.st.target_logprobs(x, targets.cuda(), topk, mask.cuda() if mask is not None else None, temperature)
    # At 1e15 and more 64 bits cannot hold a sum's logarithm beside the offset: the form takes the distances from each
    # row's largest score, and lse the offset afterwards.
    raw, allowed = logits.double(), torch.ones(logits.shape, dtype=torch.bool)
    if mask is not None:
        allowed = O.bits(mask.expand(rows, -1), columns)
    top = torch.where(allowed, raw, -math.inf).amax(1)
    leaf = torch.where(allowed, raw - top.unsqueeze(1), 0.0).requires_grad_()
    want = list(O.target_logprobs(leaf, targets, topk, mask, temperature))
    assert torch.equal(out[3].cpu(), want[3]), "top_ids"
    want_lse = want[2].detach() + top / temperature
    _near(out[2], want_lse, 64 * U * (1 + wide + want_lse.abs()), "lse")
    for i, what in ((0, "logprobs"), (4, "top_logprobs")):
        size = torch.where(torch.isfinite(want[i]), want[i].detach(), 0.0).abs()
        _near(out[i], want[i], 64 * U * (1 + wide + size), what)
    _near(out[1], want[1], 64 * U * (1 + 2 * wide), "entropy")

    g = torch.Generator().manual_seed(rows * 31 + columns)
    cot = [torch.randn(o.shape, generator=g) for o in (out[0], out[1], out[2], out[4])]
    got, = torch.autograd.grad([out[0], out[1], out[2], out[4]], [x], [c.cuda() for c in cot])
    total = sum((torch.where(torch.isfinite(w), w, 0.0) * c).sum() for w, c in zip((want[0], want[1], want[2], want[4]), cot))
    grad, = torch.autograd.grad(total, leaf)
    with torch.no_grad():
        z = torch.where(allowed, leaf / temperature, -math.inf)
        lse = want[2].unsqueeze(1)
        p = torch.where(allowed, (z - lse).exp(), 0.0)
        logp = torch.where(p > 0, z - lse, 0.0)
        whole = cot[0].abs() + cot[2].abs() + cot[3].abs().sum(1)
        terms = p * (whole.unsqueeze(1) + cot[1].abs().unsqueeze(1) * (logp.abs() + want[1].unsqueeze(1)))
        terms.scatter_add_(1, targets.clamp(0, columns - 1).unsqueeze(1), cot[0].abs().double().unsqueeze(1))
        terms.scatter_add_(1, want[3].clamp(min=0), cot[3].abs().double())
        atol = terms / temperature * (128 * U * (1 + wide + logp.abs()) + HALF[logits.dtype] * 1.01) + TINY[logits.dtype]
    _near(got, grad, atol, "grad_logits")
    assert not got.cpu()[~allowed].any()


# z / T of a row's scores: where the product with log2 e has an ulp of a hundredth, of more than one, and of more than
# the exponents of 32 bits
CENTRES = [1e3, 1e5, 3e6, 4.65e7, 1e8, 1.4e9, 1.44e9, 1.49e9, 2e9, 1e10, 1e15, 1e25]


@pytest.mark.parametrize("columns", [300, 70_001])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize("centre", [s * c for c in CENTRES for s in (1, -1)])
def test_logprobs_far_from_zero(centre, temperature, columns):
    """Rows around a large score, an ordinary one beside them, rows of both, with either sign, filtered and whole."""
    H.note(f"[logprobs] scores / T around {centre} T {temperature} columns {columns}")
    g = torch.Generator().manual_seed(columns)
    noise = torch.randn((6, columns), generator=g).double() * 2
    at = torch.arange(columns)
    z = noise.clone()
    z[0] += centre
    z[1] += torch.where(at % 2 == 0, centre, 0.0)
    z[2] += torch.where(at < columns // 2, centre, -centre)
    z[3] += torch.where(at // 8 % 5 == 0, -centre, centre)
    z[5] += centre * (1 + (at % 7) * 2.0 ** -22)
    logits = (z * temperature).float()
    targets = torch.randint(0, columns, (6,), generator=g)
    passes = torch.rand((6, columns), generator=g) < 0.4
    passes[torch.arange(6), targets] = True
    for mask in (None, O.pack(passes)):
        _check_logprobs(logits, targets, 7, mask, temperature)


@pytest.mark.parametrize("columns", [300, 70_001])
@pytest.mark.parametrize("dtype,temperature,scale", [
    (torch.float16, 1e-5, 20_000.0), (torch.float16, 1e-6, 500.0), (torch.bfloat16, 1.0, 1e12), (torch.bfloat16, 1e-3, 1e6),
    (torch.bfloat16, 1.0, 1e32), (torch.float32, 1.0, 1e9), (torch.float32, 1e-6, 1e4), (torch.float32, 1e6, 1e15)])
def test_logprobs_wide_scores(dtype, temperature, scale, columns):
    """Scores that spread over many multiples of the temperature."""
    H.note(f"[logprobs] wide scores {dtype} T {temperature} scale {scale} columns {columns}")
    g = torch.Generator().manual_seed(3)
    largest = torch.finfo(dtype).max
    logits = (torch.randn((3, columns), generator=g) * scale).clamp(-largest, largest).to(dtype)
    targets = torch.randint(0, columns, (3,), generator=g)
    targets[0] = logits[0].float().argmax()
    _check_logprobs(logits, targets, 4, None, temperature)


@pytest.mark.parametrize("temperature", [1e-6, 1.0])
@pytest.mark.parametrize("columns", [20_000, 70_001])
def test_logprobs_rise_through_large_scores(columns, temperature):
    """Scores that rise, or fall, through the large ones of either sign, a little a column: every thread meets them in
    order."""
    H.note(f"[logprobs] rising scores T {temperature} columns {columns}")
    at = torch.arange(columns).double()
    up = [c + at * (64.0 / columns) * step for c in (-4.65e7, 4.65e7, -3.3e7, 9.3e7) for step in (1, 16)]
    up += [c + at * (1e9 / columns) for c in (1e9, -2e9, -1.5e9)]
    z = torch.stack(up + [r.flip(0) for r in up])
    _check_logprobs((z * temperature).float(), torch.arange(len(z)) * 11, 3, None, temperature)


# ------------------------------------------------------------------ routing


def _route_rows(clusters, centre, dtype):
    """Rows around a large score, ordinary ones, rows of both, with either sign."""
    g = torch.Generator().manual_seed(clusters)
    z = torch.randn((9, clusters), generator=g).double() * 2
    at = torch.arange(clusters)
    z[0] += centre
    z[2] += torch.where(at % 2 == 0, centre, 0.0)
    z[4] += torch.where(at < clusters // 2, centre, -centre)
    z[5] += centre * (1 + (at % 7) * 2.0 ** -22)
    z[8] -= centre
    return z.to(dtype)


def _route_oracle(logits, probes):
    """The form of the distances from each row's largest score (what lies at the offset 64 bits cannot hold beside a
    sum's logarithm), lse with the offset; and log p."""
    top = logits.double().amax(1)
    leaf = (logits.double() - top.unsqueeze(1)).requires_grad_()
    want = list(O.cluster_route(leaf, probes))
    log_p = (leaf - want[2].unsqueeze(1)).detach()
    return leaf, want, want[2].detach() + top, log_p


ROUTE_CENTRES = [1e3, 1e5, 1e6, 1.04e6, 1.05e6, 3e6, 1e8, 1.45e9, 3e9, 1e10, 1e15, 1e25, 9e29, 2e30]


@pytest.mark.parametrize("clusters,probes", [(60, 5), (200, 16), (700, 8), (1800, 30), (3000, 12), (10_000, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("centre", [s * c for c in ROUTE_CENTRES for s in (1, -1)])
def test_route_far_from_zero(centre, dtype, clusters, probes):
    """The outputs of rows around a large score, and the loss over them and ordinary ones."""
    H.note(f"[route] scores around {centre} {dtype} clusters {clusters}")
    logits = _route_rows(clusters, centre, dtype)
    out = torch.ops.st.cluster_route(logits.cuda(), probes)
    _, want, lse, log_p = _route_oracle(logits, probes)
    wide = math.log(clusters)
    assert torch.equal(out[0].cpu(), want[0]) and torch.equal(out[3].cpu(), want[3])
    size = log_p.gather(1, want[0]).abs()
    _near(out[1], want[1], 64 * U * (1 + wide + size) * want[1].detach() + 1e-37, "weights")
    _near(out[2], lse, 64 * U * (1 + wide + lse.abs()), "lse")
    # a sum over the rows, one more rounding for each
    _near(out[4], want[4], U * (64 * (1 + 2 * wide) + len(logits)) * want[4].detach(), "loss")


@pytest.mark.parametrize("clusters,probes", [(60, 5), (200, 16), (700, 8), (1800, 30), (3000, 12), (10_000, 20)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("centre", [s * c for c in ROUTE_CENTRES for s in (1, -1)])
def test_route_gradient_far_from_zero(centre, dtype, clusters, probes):
    """The gradient of rows around a large score."""
    H.note(f"[route] gradient around {centre} {dtype} clusters {clusters}")
    logits = _route_rows(clusters, centre, dtype)
    rows, wide = len(logits), math.log(clusters)
    x = logits.cuda().requires_grad_()
    out = torch.ops.st.cluster_route(x, probes)
    leaf, want, _, log_p = _route_oracle(logits, probes)
    g = torch.Generator().manual_seed(rows)
    cot = [torch.randn(out[1].shape, generator=g), torch.randn(out[2].shape, generator=g), torch.tensor(1.7)]
    got, = torch.autograd.grad([out[1], out[2], out[4]], [x], [c.cuda() for c in cot])
    grad, = torch.autograd.grad(sum((w * c).sum() for w, c in zip((want[1], want[2], want[4]), cot)), leaf)
    p = log_p.exp()
    a = (1.7 * clusters * want[3].double() / (probes * rows * rows)).expand_as(p).clone()
    a.scatter_add_(1, want[0], cot[0].abs().double())
    terms = p * (a + (p * a).sum(1, keepdim=True) + cot[1].abs().unsqueeze(1))
    log_p = torch.where(p > 0, log_p, 0.0)
    _near(got, grad, terms * (128 * U * (1 + wide + log_p.abs()) + HALF[dtype] * 1.01) + TINY[dtype], "grad_logits")


@pytest.mark.parametrize("clusters", [60, 700, 5000])
@pytest.mark.parametrize("offset", [2.0 ** 10, 2.0 ** 16, 2.0 ** 19, 2.0 ** 20, 2.0 ** 22])
def test_gradients_without_the_offset(offset, clusters):
    """Scores of multiples of a half have gradients, of both operators, that an offset does not change: each side is
    within 128 u (1 + L + |log p|) of the terms' sizes, which are at most 2 max |cotangent| p here."""
    H.note(f"[head] offset {offset} clusters {clusters}")
    g = torch.Generator().manual_seed(5)
    z = torch.randint(-12, 12, (7, clusters), generator=g).float() / 2
    weights = torch.randn((7, 6), generator=g).cuda()
    targets = torch.randint(0, clusters, (7,), generator=g).cuda()

    def gradients(scores):
        x = scores.cuda().requires_grad_()
        route = torch.autograd.grad((torch.ops.st.cluster_route(x, 6)[1] * weights).sum(), x)[0]
        o = torch.ops.st.target_logprobs(x, targets)
        return route.cpu().double(), torch.autograd.grad(o[0].sum() + o[1].sum(), x)[0].cpu().double()

    p = torch.softmax(z.double(), 1)
    size = 128 * U * (1 + math.log(clusters) + p.log().abs())
    at = torch.zeros_like(p).scatter_(1, targets.cpu().unsqueeze(1), 1.0)
    entropy = -(p * p.log()).sum(1, keepdim=True)
    for (a, b), terms in zip(zip(gradients(z), gradients(z + offset)),
                             (2 * p * weights.abs().max().item(), at + p * (1 + p.log().abs() + entropy))):
        _near(b.float(), a, 2 * size * terms + 1e-37)


# ------------------------------------------------------------------ 4-bit tables


@pytest.mark.parametrize("group_size", [1 << 21, 1 << 40, (1 << 63) - 32])
def test_group_sizes_past_the_columns(group_size):
    """One group, as of the first multiple of 32 that holds the columns."""
    H.note(f"[int4] group size {group_size}")
    g = torch.Generator().manual_seed(2)
    for dim in (1, 31, 32, 40, 300):
        w, x = torch.randn((70, dim), generator=g).cuda(), torch.randn((3, dim), generator=g).cuda()
        least = -(-dim // 32) * 32
        for symmetric in (True, False):
            want = torch.ops.st.int4_quantize(w, least, symmetric)
            got = torch.ops.st.int4_quantize(w, group_size, symmetric)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert torch.equal(torch.ops.st.int4_matvec(*got[:2], x, group_size, got[2]),
                               torch.ops.st.int4_matvec(*want[:2], x, least, want[2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_differences_past_the_type(dtype):
    """A group from -3e38 to 3e38 has a finite scale, (hi - lo) / 15 to its type's rounding (a rounding of each of two
    quotients and of their difference before that), and codes within half a step of the weights (the zero point is
    rounded to a whole code, and so are the weights: one step at most)."""
    H.note(f"[int4] wide groups {dtype}")
    w = (torch.randn((6, 96), generator=torch.Generator().manual_seed(4)) * 1e38).clamp(-3.3e38, 3.3e38)
    w[0, :2] = torch.tensor([3.3e38, -3.3e38])
    w[1, 40:42] = torch.tensor([-2.9e38, 1.2e38])
    w[2] = 3.3e38
    w[3, ::3] = -3.3e38
    w = w.to(dtype)
    packed, scales, zeros = (t.cpu() for t in torch.ops.st.int4_quantize(w.cuda(), 32, False))
    groups = w.double().view(6, 3, 32)
    lo, hi = groups.amin(2).clamp(max=0), groups.amax(2).clamp(min=0)
    want = (hi - lo) / 15
    _near(scales, want, want * (4 * U + HALF[dtype] * 1.01), "scales")
    back = O.dequantize(packed, scales, zeros, 96, 32)
    assert ((back - w.double()).abs() <= scales.double().repeat_interleave(32, 1) * 1.01 + want.repeat_interleave(32, 1) * 15 * HALF[dtype]).all()


def test_matvec_bits_of_each_element():
    """What a product keeps of its vector's elements.  Rows of one code of 1 and scale 1 give the elements back: of
    float32 vectors each to 2^-23 of itself, at and beside elements 2^27 times as large, and below that to 2^-50 of the
    largest; of bfloat16 ones exactly down to 2^-31 of the largest, to 2^-39 of it below; float16 ones exactly."""
    H.note("[int4] bits of each element")
    dim = 256
    codes = torch.full((dim, dim), 8, dtype=torch.uint8)
    codes.fill_diagonal_(9)
    packed = (codes[:, ::2] | (codes[:, 1::2] << 4)).cuda()
    scales = torch.ones((dim, dim // 32)).cuda()
    g = torch.Generator().manual_seed(8)

    def kept(x):
        return torch.ops.st.int4_matvec(packed, scales, x.cuda(), 32, None, torch.float32).cpu().double()

    for size in (1.0, 2.0 ** 100, 2.0 ** -100):
        for low in (0, -10, -27, -40, -60):
            x = (1 + torch.rand((40, dim), generator=g)) * torch.where(torch.rand((40, dim), generator=g) < 0.5, 1.0, -1.0)
            x *= torch.exp2(torch.randint(low, 1, (40, dim), generator=g).float()) * size
            x[:, 0] = 1.9999 * size
            largest = x.double().abs().amax(1, keepdim=True)
            _near(kept(x).float(), x, torch.maximum(x.double().abs() * 2.0 ** -23, largest * 2.0 ** -50), low)
            b = x.bfloat16()
            largest = b.double().abs().amax(1, keepdim=True)
            near = b.double().abs() >= largest * 2.0 ** -31
            _near(kept(b).float(), b.double(), torch.where(near, 0.0, largest * 2.0 ** -39), low)
            # the whole of a float32 vector, as two vectors
            if low >= -10:
                top = x.bfloat16().float()
                assert torch.equal(kept(top) + kept(x - top), x.double())
    h = torch.randint(-32768, 32768, (40, dim), generator=g, dtype=torch.int16).view(torch.float16)
    h = torch.where(torch.isfinite(h), h, torch.ones_like(h))
    assert torch.equal(kept(h), h.double())
