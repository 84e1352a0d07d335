"""Queries over the 4-bit cache: elements of very different sizes, and each type held
to what its arithmetic gives.

Tolerances (relative 2-norm).  Weights are rounded to fp16 whatever the type
(2^-12 at most an element, half that in the mean), and scores carry 1e-4 of |q| times a
code unit, 5e-5 of a weight here.  So an fp16 output, itself rounded by 2^-12 at
most, is within 2^-11, and a bf16 output within its own rounding, 2^-9 at most,
and half as much for the rest: 2^-8 as elsewhere."""
import pytest
import torch

import tda_b200
from tests.sdiff_reference import decode64, rel
from tests.test_gpu_cache4 import expected, filled

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def cache_of(n, D, Hkv, dtype, seed, normalize, page=32):
    """n tokens whose keys are zero in their first group of 32."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = tda_b200.Cache4(-(-n // page), page, Hkv, D, normalize_keys=normalize)
    u = 0.6 * torch.randn(2, Hkv, D, generator=g, device=DEV)
    kv = [torch.randn(n, Hkv, D, generator=g, device=DEV) for _ in range(3)]
    for i in range(2):
        kv[i] += u[i]
        kv[i][..., :32] = 0
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    tda_b200.cache4_append(cache, *(t.to(dtype) for t in kv), slots)
    table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None]
    return cache, table, torch.tensor([n], dtype=torch.int32, device=DEV), slots, u, g


@pytest.mark.parametrize("dtype,large", [(torch.float16, 30000.0), (torch.float16, 1000.0), (torch.bfloat16, 2e6), (torch.bfloat16, 2e4)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [50, 600])
def test_one_element_far_above_the_others(dtype, large, D, n):
    """It meets keys of zero: the score is that of the small elements, to their own precision."""
    H, Hkv = 4, 2
    cache, table, lengths, slots, u, g = cache_of(n, D, Hkv, dtype, D, False)
    q = [torch.randn(1, H, D, generator=g, device=DEV).to(dtype) for _ in range(2)]
    for t in q:
        t[..., 3] = large
    lam = torch.full((H,), 0.4, device=DEV)
    out = tda_b200.cache4_softmax_attention(*q, cache, table, lengths, 0.4)
    want = decode64(q[0][0], q[1][0], *tda_b200.cache4_read(cache, slots, torch.float32), lam)
    assert rel(out[0], want) <= TOL[dtype], rel(out[0], want)


def test_queries_of_zero():
    """Every key has the same weight."""
    n, H = 300, 4
    for dtype in (torch.float16, torch.bfloat16):
        cache, table, lengths, slots, _, g = cache_of(n, 128, 2, dtype, 1, False)
        q = torch.zeros(1, H, 128, dtype=dtype, device=DEV)
        v = tda_b200.cache4_read(cache, slots, torch.float32)[2].double().mean(0).repeat_interleave(2, 0)
        out = tda_b200.cache4_softmax_attention(q, q, cache, table, lengths, 0.25)
        assert rel(out[0], 0.75 * v) <= TOL[dtype]


@pytest.mark.parametrize("D,page,H,Hkv", [(64, 32, 4, 4), (128, 64, 8, 2), (128, 16, 5, 1)])
def test_fp16_softmax_form(D, page, H, Hkv):
    lens = [1, 17, 64, 300, 2500]
    cache, table, lengths, slots, q1, q2 = filled(lens, H, Hkv, D, page, torch.float16, H)
    lam = torch.linspace(-0.5, 0.7, H, device=DEV)
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, lam.reshape(1, H, 1, 1))
    want = expected(cache, slots, q1, q2, lam)
    for b in range(len(lens)):
        assert rel(out[b], want[b]) <= TOL[torch.float16], (lens[b], rel(out[b], want[b]))


@pytest.mark.parametrize("D,page,H,Hkv", [(64, 32, 4, 4), (128, 64, 8, 2), (128, 16, 5, 1)])
@pytest.mark.parametrize("power", [1.0, 2.0, 3.0, 1.5])
def test_fp16_threshold_form(D, page, H, Hkv, power):
    """Weights keep their rounding rest here; scores are exact products summed in fp32, 2^-20 of |q| |k|, against
    a threshold near which a weight p z^(p-1) small adds little."""
    lens = [64, 300, 2500]
    cache, table, lengths, slots, q1, q2 = filled(lens, H, Hkv, D, page, torch.float16, H + 1, True, lean=0.6)
    lam = torch.linspace(0.0, 0.7, H, device=DEV)
    out = tda_b200.cache4_threshold_attention(q1, q2, cache, table, lengths, 0.9, lam.reshape(H, 1, 1), power)
    want = expected(cache, slots, q1, q2, lam, threshold=True, beta=0.9, power=power)
    for b in range(len(lens)):
        assert rel(out[b], want[b]) <= TOL[torch.float16] or float((out[b].double() - want[b]).abs().max()) <= 1e-6, \
            (lens[b], rel(out[b], want[b]))
