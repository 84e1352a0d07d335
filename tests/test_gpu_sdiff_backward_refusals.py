"""sdiff_backward reads dout, o12 and lse by pointer: what does not fit raises before a launch."""
import pytest
import torch

import tda_b200

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def call():
    q = torch.randn(2, 4, 70, 64, device="cuda").to(torch.bfloat16)
    k = torch.randn(2, 2, 90, 64, device="cuda").to(torch.bfloat16)
    out, o12, lse = tda_b200.sdiff_forward(q, q, k, k, k, 0.5)
    return [q, q, k, k, k], dict(dout=out, o12=o12, lse=lse)


@pytest.mark.parametrize("name,change,error", [
    ("dout", lambda t: None, TypeError), ("dout", lambda t: t[:, :, :69], ValueError), ("dout", lambda t: t.cpu(), RuntimeError),
    ("dout", lambda t: t.int(), TypeError),
    ("o12", lambda t: None, TypeError), ("o12", lambda t: t[:1], ValueError), ("o12", lambda t: t[..., :32], ValueError),
    ("o12", lambda t: t.to(torch.bfloat16), TypeError), ("o12", lambda t: t.cpu(), RuntimeError),
    ("o12", lambda t: t.transpose(3, 4).contiguous().transpose(3, 4), TypeError),
    ("lse", lambda t: None, TypeError), ("lse", lambda t: t[0], ValueError), ("lse", lambda t: t.double(), TypeError),
    ("lse", lambda t: t.cpu(), RuntimeError), ("lse", lambda t: t.expand(2, 2, 4, 70)[:, :, :, :1].expand(2, 2, 4, 70), TypeError),
])
def test_refusals(call, name, change, error):
    xs, kw = call
    with pytest.raises(error, match=name):
        tda_b200.sdiff_backward(*xs, **{**kw, name: change(kw[name])}, lambda_param=0.5)


def test_a_gradient_of_another_type_and_layout(call):
    xs, kw = call
    a = tda_b200.sdiff_backward(*xs, **kw, lambda_param=0.5)
    wide = kw["dout"].float().transpose(1, 2).contiguous().transpose(1, 2)
    b = tda_b200.sdiff_backward(*xs, **{**kw, "dout": wide}, lambda_param=0.5)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
