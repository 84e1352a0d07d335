"""4-bit cache attention where values are zero or tiny, and fp16 queries held to
what their arithmetic gives."""
import pytest
import torch

import tda_b200
from tests.sdiff_reference import decode64, rel

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.0 ** -8  # bf16: the output's rounding, 2^-9, and half as much for all else


def build(n, dtype, seed, values, normalize=True, H=4, Hkv=2, D=128, page=64):
    """One request of n tokens whose value rows are scaled by ``values`` (n,)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = tda_b200.Cache4(n // page + 1, page, Hkv, D, normalize_keys=normalize)
    table = torch.arange(n // page + 1, dtype=torch.int32, device=DEV)[None]
    u = 0.6 * torch.randn(2, Hkv, D, generator=g, device=DEV)
    k = [(torch.randn(n, Hkv, D, generator=g, device=DEV) + u[i]).to(dtype) for i in range(2)]
    v = (torch.randn(n, Hkv, D, generator=g, device=DEV) * values[:, None, None]).to(dtype)
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    tda_b200.cache4_append(cache, *k, v, slots)
    lift = u.repeat_interleave(H // Hkv, 1)
    q = [(torch.randn(1, H, D, generator=g, device=DEV) + lift[i]).to(dtype) for i in range(2)]
    return cache, table, torch.tensor([n], dtype=torch.int32, device=DEV), slots, q


def held(cache, slots):
    return tda_b200.cache4_read(cache, slots, torch.float32)


@pytest.mark.parametrize("power", [1.0, 2.0, 4.0, 8.0])
@pytest.mark.parametrize("n", [40, 700, 9000])
def test_threshold_form_over_values_of_zero(power, n):
    """All zero, zero in front, and a single row that is not."""
    lam = torch.full((4,), 0.4, device=DEV)
    ones = torch.ones(n, device=DEV)
    lone = torch.zeros(n, device=DEV)
    lone[n - 3] = 1.0
    for values in (0 * ones, torch.where(torch.arange(n, device=DEV) < n // 2, 0.0, 1.0), lone):
        cache, table, lengths, slots, q = build(n, torch.bfloat16, n, values)
        out = tda_b200.cache4_threshold_attention(*q, cache, table, lengths, 0.9, 0.4, power)
        want = decode64(q[0][0], q[1][0], *held(cache, slots), lam, True, 0.9, power, True)
        assert torch.isfinite(out).all()
        assert rel(out[0], want) <= TOL or float((out[0].double() - want).abs().max()) <= 1e-5 * float(want.abs().max()), rel(out[0], want)


@pytest.mark.parametrize("n", [40, 700, 9000])
def test_weights_next_to_the_threshold(n):
    """beta so large that only the best keys pass, by little: weights of 1e-12 and less over values of zero."""
    cache, table, lengths, slots, q = build(n, torch.bfloat16, n, torch.zeros(n, device=DEV))
    for beta in torch.linspace(0.5, 4.0, 15).tolist():
        out = tda_b200.cache4_threshold_attention(*q, cache, table, lengths, beta, 0.4, 4.0)
        assert float(out.abs().max()) == 0.0, beta


@pytest.mark.parametrize("first,rest", [(0.0, 1.0), (0.0, 1e-6), (0.0, 1e-20), (1e-20, 1.0), (1.0, 0.0), (1e-20, 1e-20)])
@pytest.mark.parametrize("n", [100, 900, 9000])
def test_softmax_form_over_values_of_any_size(first, rest, n):
    """The output is as exact as its values' size allows, whatever stands in front of them."""
    values = torch.where(torch.arange(n, device=DEV) < n // 2, first, rest)
    cache, table, lengths, slots, q = build(n, torch.bfloat16, n + 1, values, normalize=False)
    out = tda_b200.cache4_softmax_attention(*q, cache, table, lengths, 0.4)
    want = decode64(q[0][0], q[1][0], *held(cache, slots), torch.full((4,), 0.4, device=DEV))
    assert rel(out[0], want) <= TOL, rel(out[0], want)
