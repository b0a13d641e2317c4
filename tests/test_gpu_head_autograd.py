"""What the retrieval head's operators do with gradients they do not have."""

import warnings

import pytest
import torch

from tests import gpu_helpers as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")
    import silvertorch_amd.ops._load_ops  # noqa: F401


def _refuses(message, call):
    with pytest.raises(RuntimeError, match=message):
        call()


@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_four_bit_products_refuse_gradients(device):
    """A result that depends on vectors or scales which require a gradient is computed as ever, and says that it has no
    gradient when one is asked for; so does the table's making."""
    H.note(f"[head] int4 gradients {device}")
    g = torch.Generator().manual_seed(1)
    packed, scales, zeros = torch.ops.st.int4_quantize(torch.randn((40, 70), generator=g).to(device), 32)
    x = torch.randn((3, 70), generator=g).to(device)
    want = torch.ops.st.int4_matvec(packed, scales, x, 32, zeros)
    assert not want.requires_grad
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for xs, ss in ((x.clone().requires_grad_(), scales), (x, scales.clone().requires_grad_())):
            y = torch.ops.st.int4_matvec(packed, ss, xs, 32, zeros)
            assert torch.equal(y.detach(), want)
            _refuses("int4_matvec has no gradient", lambda: y.sum().backward())
            y = torch.ops.st.int4_matvec(packed, ss, xs, 32, zeros)
            y.mul_(2)  # results may be changed in place, as any operator's
            _refuses("int4_matvec has no gradient", lambda: y.sum().backward())
            with torch.no_grad():
                assert not torch.ops.st.int4_matvec(packed, ss, xs, 32, zeros).requires_grad
        w = torch.randn((5, 64), generator=g).to(device)
        plain = torch.ops.st.int4_quantize(w, 32)
        made = torch.ops.st.int4_quantize(w.clone().requires_grad_(), 32)
        assert all(torch.equal(a.detach(), b) for a, b in zip(made, plain))
        assert not made[0].requires_grad and not made[2].requires_grad
        _refuses("int4_quantize has no gradient", lambda: made[1].sum().backward())


def test_module_refuses_to_train_through_its_table():
    """A query tower is not tuned against a packed table: the loss says so."""
    H.note("[head] module gradients")
    from silvertorch_amd.modules import RetrievalHeadModule

    torch.manual_seed(0)
    docs = torch.nn.Parameter(torch.randn((500, 64), device="cuda"))
    tower = torch.nn.Linear(16, 64, device="cuda")
    head = RetrievalHeadModule(group_size=32, topk=3, temperature=0.5)
    head.set_embeddings(docs)
    assert not any(b.requires_grad for b in head.buffers())
    q = torch.randn((4, 16), device="cuda")
    logprobs, _, _, ids, _ = head(tower(q), torch.arange(4, device="cuda"))
    with torch.no_grad():
        again = head(tower(q), torch.arange(4, device="cuda"))
    assert torch.equal(logprobs.detach(), again[0]) and torch.equal(ids, again[3])
    _refuses("int4_matvec has no gradient", lambda: (-logprobs.mean()).backward())
    assert all(p.grad is None for p in tower.parameters())


def test_tangents_are_refused():
    """An input with a forward-mode tangent is refused; beside one, and with forward mode off, calls are as ever."""
    H.note("[head] tangents")
    import torch.autograd.forward_ad as fwAD

    z = torch.randn((3, 300), generator=torch.Generator().manual_seed(1)).cuda()
    targets = torch.arange(3, device="cuda")
    packed, scales, zeros = torch.ops.st.int4_quantize(z, 32)
    calls = {
        "target_logprobs": lambda t: torch.ops.st.target_logprobs(t, targets, 4),
        "cluster_route": lambda t: torch.ops.st.cluster_route(t, 4),
        "int4_matvec": lambda t: (torch.ops.st.int4_matvec(packed, scales, t, 32, zeros),),
        "int4_quantize": lambda t: torch.ops.st.int4_quantize(t, 32),
    }
    for name, call in calls.items():
        want = call(z)
        with fwAD.dual_level():
            dual = fwAD.make_dual(z, torch.ones_like(z))
            _refuses(f"{name} has no forward-mode derivative", lambda: call(dual))
            with fwAD._set_fwd_grad_enabled(False):
                assert all(torch.equal(a, b) for a, b in zip(call(dual), want))
            assert all(torch.equal(a, b) for a, b in zip(call(fwAD.unpack_dual(dual).primal), want))
