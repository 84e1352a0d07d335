"""differential_softmax_attention traces without a GPU, as the threshold functions do."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import tda_b200

SHAPES = [(2, 4, 7, 64)] * 2 + [(2, 2, 9, 64)] * 3


def on_meta():
    return [torch.empty(s, dtype=torch.bfloat16, device="meta") for s in SHAPES]


def test_fake_tensors():
    with FakeTensorMode():
        xs = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in SHAPES]
        for lam in (0.5, torch.empty(1, 4, 1, 1, device="cuda")):
            out = tda_b200.differential_softmax_attention(*xs, lam)
            assert out.shape == SHAPES[0] and out.dtype == torch.bfloat16


def test_meta_tensors_and_their_gradients():
    xs = [x.requires_grad_(True) for x in on_meta()]
    lam = torch.empty(1, 4, 1, 1, device="meta", requires_grad=True)
    out = tda_b200.differential_softmax_attention(*xs, lam)
    assert out.shape == SHAPES[0] and out.is_meta
    grads = torch.autograd.grad(out, xs + [lam], torch.empty_like(out))
    assert [g.shape for g in grads] == [x.shape for x in xs] + [lam.shape]


def test_make_fx():
    graph = make_fx(lambda *a: tda_b200.differential_softmax_attention(*a, 0.5), tracing_mode="fake")(*on_meta())
    assert any("sdiff_fwd" in str(n.target) for n in graph.graph.nodes)


@pytest.mark.parametrize("grad", [False, True])
def test_compile_fullgraph(grad):
    torch._dynamo.reset()
    fn = torch.compile(lambda *a: tda_b200.differential_softmax_attention(*a), fullgraph=True, backend="aot_eager")
    xs = [x.requires_grad_(grad) for x in on_meta()]
    out = fn(*xs, 0.5)
    assert out.shape == SHAPES[0]
    if grad:
        out.float().sum().backward()
        assert all(x.grad.shape == x.shape for x in xs)


def saved_shapes(fn, xs):
    """Shapes of the operator's outputs in the graph that torch.compile makes of fn."""
    seen = []

    def backend(gm, _example):
        seen.extend(tuple(t.shape for t in n.meta["example_value"]) for n in gm.graph.nodes if "sdiff_fwd" in str(n.target))
        return gm.forward

    torch._dynamo.reset()
    torch.compile(fn, fullgraph=True, backend=backend)(*xs)
    return seen


def test_compiled_inference_keeps_nothing_for_a_backward():
    """o12 and lse are four times the output's bytes."""
    fn = lambda *a: tda_b200.differential_softmax_attention(*a, 0.5)
    xs = on_meta()
    assert saved_shapes(fn, xs) == [(SHAPES[0], (0,), (0,))]
    wants = [x.requires_grad_(True) for x in on_meta()]
    assert saved_shapes(fn, wants) == [(SHAPES[0], (2, *SHAPES[0]), (2, *SHAPES[0][:3]))]
    with torch.no_grad():
        assert saved_shapes(fn, wants) == [(SHAPES[0], (0,), (0,))]
