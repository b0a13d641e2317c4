"""The query tower's differentiable operators go through the dispatcher, with
and without gradients: a dispatch mode sees each kernel's operator (and may
answer in its place, which is how these tests run without a GPU), and a fake
tensor does not reach a kernel.  Refusals of the operators that the gradients
call."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

import silvertorch_amd.ops._load_ops  # noqa: F401

st = torch.ops.st


class Answers(TorchDispatchMode):
    """Names of st operators, answered with tensors of ones of the right shapes."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace != "st":
            return func(*args, **(kwargs or {}))
        name = func._schema.name.removeprefix("st::")
        self.seen.append(name)
        if name == "dropout":
            return torch.ones_like(args[0])
        if name == "dropout_with_state":
            return torch.ones_like(args[0]), args[2].clone()
        if name == "layer_norm":
            return torch.ones_like(args[0])
        if name == "layer_norm_with_stats":
            return torch.ones_like(args[0]), torch.ones((args[0].numel() // args[0].shape[-1], 3))
        if name == "dropout_add_layer_norm":
            return torch.ones_like(args[0]), torch.ones_like(args[1])
        if name == "dropout_add_layer_norm_with_stats":
            used = args[5].clone() if len(args) > 5 and args[5] is not None and args[4] > 0 else None
            return torch.ones_like(args[0]), torch.ones_like(args[1]), torch.ones((len(args[0]), 3)), used
        assert name == "layer_norm_backward"
        grad_y, grad_sum, h, weight, stats, used, p, y_type, weight_type, wanted = args
        self.wanted = list(wanted)
        self.used = used
        sizes = [h.shape, h.shape, h.shape[-1:], h.shape[-1:]]
        types_ = [y_type, h.dtype, weight_type, weight_type]
        return tuple(torch.full(s, 2.0, dtype=t) if on else None for s, t, on in zip(sizes, types_, wanted))


def _inputs(grad, dtype=torch.float32):
    x, res = torch.ones((3, 40), dtype=dtype), torch.ones((3, 40))
    w, b = torch.ones(40), torch.ones(40)
    return [t.requires_grad_(grad) for t in (x, res, w, b)], torch.tensor([1, 2])


@pytest.mark.parametrize("grad", [False, True])
def test_a_mode_sees_dropout(grad):
    (x, *_), s = _inputs(grad)
    with Answers() as mode:
        y = st.dropout(x, 0.5, s)
        if grad:
            g, = torch.autograd.grad(y.sum(), x)
            assert torch.equal(g, torch.ones_like(x))
    assert mode.seen == (["dropout_with_state", "dropout"] if grad else ["dropout"])


@pytest.mark.parametrize("grad", [False, True])
def test_a_mode_sees_layer_norm(grad):
    (x, _, w, b), _ = _inputs(grad)
    with Answers() as mode:
        y = st.layer_norm(x, w, b)
        if grad:
            assert all((g == 2).all() for g in torch.autograd.grad(y.sum(), [x, w, b]))
    assert mode.seen == (["layer_norm_with_stats", "layer_norm_backward"] if grad else ["layer_norm"])
    if grad:
        assert mode.wanted == [True, False, True, True]


@pytest.mark.parametrize("wanted", [[True, True, True, True], [True, False, False, False], [False, True, False, True],
                                    [False, False, True, False]])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_a_mode_sees_dropout_add_layer_norm(wanted, p):
    leaves, s = _inputs(False, torch.bfloat16)
    for t, on in zip(leaves, wanted):
        t.requires_grad_(on)
    x, res, w, b = leaves
    with Answers() as mode:
        y, total = st.dropout_add_layer_norm(x, res, w, b, p, s)
        grads = torch.autograd.grad(y.sum(), [t for t, on in zip(leaves, wanted) if on])
    assert mode.seen == ["dropout_add_layer_norm_with_stats", "layer_norm_backward"] and mode.wanted == wanted
    assert (mode.used is not None) == (p > 0)
    assert [g.dtype for g in grads] == [t.dtype for t, on in zip(leaves, wanted) if on] and all((g == 2).all() for g in grads)
    with torch.no_grad(), Answers() as mode:
        st.dropout_add_layer_norm(x, res, w, b, p, s)
    assert mode.seen == ["dropout_add_layer_norm"]


@pytest.mark.parametrize("grad", [False, True])
def test_fake_tensors_do_not_reach_a_kernel(grad):
    mode = FakeTensorMode()
    (x, res, w, b), s = _inputs(grad)
    with mode:
        x, res, w, b, s = (mode.from_tensor(t) for t in (x, res, w, b, s))
        for call in (lambda: st.dropout(x, 0.5, s), lambda: st.layer_norm(x, w, b),
                     lambda: st.dropout_add_layer_norm(x, res, w, b, 0.5, s)):
            with pytest.raises(Exception, match=r"st\.|st::"):
                call()


def test_backward_operator_refusals():
    h, stats, w, s = torch.zeros((3, 10)), torch.zeros((3, 3)), torch.ones(10), torch.zeros(2, dtype=torch.long)
    f32 = torch.float32

    def refused(message, grad_y=h, grad_sum=None, h=h, weight=w, stats=stats, used=None, p=0.0, y_type=f32, weight_type=f32):
        with pytest.raises(RuntimeError, match=message):
            st.layer_norm_backward(grad_y, grad_sum, h, weight, stats, used, p, y_type, weight_type, [True] * 4)

    refused("shape", grad_y=h[:2])
    refused("shape", grad_sum=torch.zeros((3, 9)))
    refused("one entry", weight=w[:9])
    refused("between 1 and 32768", h=torch.zeros((3, 0)))
    refused("float32, float16 or bfloat16", h=h.double())
    refused("float32, float16 or bfloat16", y_type=torch.float64)
    refused("float32, float16 or bfloat16", weight_type=torch.int64)
    refused("x's type or float32", h=h.half(), y_type=torch.bfloat16)
    refused("stats must be", stats=stats[:2])
    refused("stats must be", stats=stats[:, :2])
    refused("stats must be", stats=stats.double())
    refused("needs the state", p=0.5)
    refused("seed and offset", p=0.5, used=s[:1])
    refused(r"p must be in \[0, 1\]", p=1.5, used=s)
    with pytest.raises(RuntimeError, match="seed and offset"):
        st.dropout_with_state(h, 0.5, s.int())
    with pytest.raises(RuntimeError, match="one entry"):
        st.layer_norm_with_stats(h, w[:9], None, 1e-5)
    with pytest.raises(RuntimeError, match="needs a state"):
        st.dropout_add_layer_norm_with_stats(h, h, None, None, 0.5, None, 1e-5)
