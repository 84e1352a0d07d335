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
