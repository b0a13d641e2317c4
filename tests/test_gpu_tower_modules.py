"""The query tower's modules on the GPU: a training pass against plain layers in
64 bits with the same dropped elements, its capture, the packed tower and the
8-bit head, the example.

Tolerances: a pass is a chain of at most 7 products of at most 128 columns each
way, each off by at most 128 u = 2^-17 of its sum of magnitudes, which is below 8
times the sum's size (2-norm) here: 14 x 8 x 2^-17 < 2^-10 of a result's 2-norm.
In 8 bits a product's operands are each off by up to half a step of max / 127,
uniformly: for rows whose largest element is 4 times their deviation or less,
4 / 127 / sqrt(12) = 0.9 % of it for either operand, 1.3 % together, 4 % over 7
products; 10 % is the bound."""

import importlib.util
from pathlib import Path

import pytest
import torch

from tests import gpu_helpers as H
from tests import tower_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _tower(**kwargs):
    from silvertorch_amd.modules import QueryTowerModule

    torch.manual_seed(0)
    tower = QueryTowerModule(24, 32, 64, layers=2, expand=2, dropout=0.3, seed=5, **kwargs).cuda()
    with torch.no_grad():
        for w, b in zip(tower.norm_weights, tower.norm_biases):
            w.add_(0.1 * torch.randn_like(w))
            b.add_(0.1 * torch.randn_like(b))
    return tower


def _plain(tower, x, rng):
    """The tower in 64 bits on the CPU with parameters of its own; rng: dropout's state ahead of the pass, None without."""
    params = {k: v.detach().cpu().double().requires_grad_() for k, v in tower.named_parameters()}
    lin = lambda name, t: t @ params[name + ".weight"].t() + params[name + ".bias"]  # noqa: E731
    place = iter(range(3))

    def drop(t):
        if rng is None:
            return t
        state = [rng[0], rng[1] + next(place)]
        return torch.where(O.keeps(t.shape, 0.3, state), t * O.times(0.3), 0.0)

    h = lin("enter", drop(x.cpu().double()))
    y = O.layer_norm(h, params["norm_weights.0"], params["norm_biases.0"])
    for i in (1, 2):
        h = h + drop(lin(f"down.{i - 1}", torch.relu(lin(f"up.{i - 1}", y))))
        y = O.layer_norm(h, params[f"norm_weights.{i}"], params[f"norm_biases.{i}"])
    return lin("leave", y), params


def _close(got, want, share):
    got, want = got.detach().cpu().double(), want.detach().double()
    assert (got - want).norm() <= share * want.norm(), ((got - want).norm() / want.norm()).item()


def test_training_pass():
    """Two passes: embeddings and every parameter's gradient, other elements dropped each time; none in evaluation."""
    H.note("[tower] module training")
    tower = _tower()
    x = torch.randn((50, 24), generator=torch.Generator().manual_seed(1)).cuda()
    g = torch.randn((50, 32), generator=torch.Generator().manual_seed(2))
    for turn in range(2):
        assert tower.rng.tolist() == [5, 3 * turn]
        out = tower(x)
        grads = torch.autograd.grad(out, list(tower.parameters()), g.cuda())
        want, params = _plain(tower, x, [5, 3 * turn])
        _close(out, want, 2.0 ** -10)
        wants = torch.autograd.grad(want, list(params.values()), g.double())
        for name, a, b in zip(params, grads, wants):
            _close(a, b, 2.0 ** -10)
    tower.eval()
    _close(tower(x), _plain(tower, x, None)[0], 2.0 ** -10)
    assert tower.rng.tolist() == [5, 6]


def test_training_pass_in_a_graph():
    """Every replay drops other elements, as eager passes from the same state do."""
    H.note("[tower] module graph")
    tower = _tower()
    x = torch.randn((50, 24), generator=torch.Generator().manual_seed(1)).cuda()
    params = list(tower.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(tower(x).square().sum(), params)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tower(x)
        grads = torch.autograd.grad(out.square().sum(), params)
        kept = [out.detach(), *grads]
    del out, grads
    start = tower.rng[1].item()
    seen = []
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        after = tower.rng.clone()
        tower.rng[1] -= 3
        assert tower.rng[1].item() == start + 3 * turn
        eager = tower(x)
        want = [eager.detach(), *torch.autograd.grad(eager.square().sum(), params)]
        assert torch.equal(tower.rng, after)
        # library products may differ in their sums' order between a graph and eager calls
        for a, b in zip(got, want):
            _close(a, b.cpu(), 2.0 ** -10)
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_packed_tower_and_head():
    """The packed tower near the trained one, in float32 and bfloat16; the 8-bit head's scores of its queries."""
    H.note("[tower] packed")
    from silvertorch_amd.modules import PackedQueryTowerModule, QueryTowerModule, RetrievalHeadModule

    torch.manual_seed(1)
    tower = QueryTowerModule(48, 64, 128, layers=2).cuda().eval()
    packed = PackedQueryTowerModule(tower)
    x = torch.randn((70, 48), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        want = tower(x)
        _close(packed(x), want.cpu(), 0.1)
        _close(packed(x[3]), want[3].cpu(), 0.1)
        assert torch.equal(packed(x.view(7, 10, 48)), packed(x).view(7, 10, 64))
        scales = packed.enter.scales.clone()
        half = PackedQueryTowerModule(tower).bfloat16()
        assert torch.equal(half.enter.scales, scales) and half.norm_weight0.dtype == torch.bfloat16
        _close(half(x.bfloat16()), want.cpu(), 0.1)
        again = PackedQueryTowerModule(QueryTowerModule(48, 64, 128, layers=2).cuda())
        again.load_state_dict(packed.state_dict())
        assert torch.equal(again(x), packed(x))
        docs = torch.randn((3001, 64), generator=torch.Generator().manual_seed(2)).cuda()
        head = RetrievalHeadModule(topk=5, temperature=0.5, bits=8)
        head.set_embeddings(docs)
        q = packed(x)
        scores = head.scores(q)
        codes, x_scales = O.codes(q.cpu())
        table, t_scales = O.codes(docs.cpu())
        exact = O.matmul(table, t_scales, codes, x_scales)
        assert ((scores.cpu().double() - exact).abs() <= 5 * 2.0 ** -24 * exact.abs() + 1e-37).all()
        logprobs, _, lse, ids, top = head(q, torch.arange(70, device="cuda"))
        order = torch.ops.st.target_logprobs(scores, torch.arange(70, device="cuda"), 5, None, 0.5)
        assert torch.equal(ids, order[3]) and torch.equal(logprobs, order[0])
    tower.requires_grad_(True)
    with pytest.raises(RuntimeError, match="int8_matmul has no gradient"):
        packed(x.clone().requires_grad_()).sum().backward()


def test_example():
    """It runs, and its loss's gradients are those of the same loss in plain operations."""
    H.note("[tower] example")
    path = Path(__file__).resolve().parents[1] / "examples" / "query_tower.py"
    spec = importlib.util.spec_from_file_location("query_tower_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    out = module.main(["--docs", "600", "--pairs", "64", "--steps", "3"])
    assert out["top_ids"].shape == (8, 5) and torch.isfinite(out["logprobs"]).all()
    tower, docs, queries, clicked = out["tower"], out["documents"], out["queries"], out["clicked"]
    tower.train()
    tower.dropout = 0.0
    got = torch.autograd.grad(module.loss_of(tower, docs, queries, clicked, 0.5), list(tower.parameters()))
    h = tower.enter(queries)
    norm = lambda t, i: torch.nn.functional.layer_norm(t, t.shape[-1:], tower.norm_weights[i], tower.norm_biases[i], tower.eps)  # noqa: E731
    y = norm(h, 0)
    for i, (up, down) in enumerate(zip(tower.up, tower.down), 1):
        h = h + down(torch.relu(up(y)))
        y = norm(h, i)
    plain = torch.nn.functional.cross_entropy(tower.leave(y) @ docs.t() / 0.5, clicked)
    for a, b in zip(got, torch.autograd.grad(plain, list(tower.parameters()))):
        _close(a, b.cpu(), 2.0 ** -10)
