"""fp32 rows in the 4-bit cache: codes equal the definition, round(7 x / amax)
with halves to even, also where x is a rounding away from a half."""
import pytest
import torch

import tda_b200
from tests.sdiff_reference import quantise64, values64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-30, 1e30])
def test_next_to_a_half(D, size):
    T, H = 4096, 2
    g = torch.Generator(device=DEV).manual_seed(D)
    top = (torch.rand(T, H, D // 32, 1, generator=g, device=DEV) + 0.5) * size
    half = torch.randint(0, 7, (T, H, D // 32, 32), generator=g, device=DEV) + 0.5
    x = (half.double() * top.double() / 7.0).float()  # the fp32 number nearest to a half
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g, device=DEV, dtype=torch.int32)).view(torch.float32)
    x = x * (1 - 2 * torch.randint(0, 2, x.shape, generator=g, device=DEV))
    x[..., 5:6] = top
    x = x.reshape(T, H, D)
    cache = tda_b200.Cache4(T // 64, 64, H, D)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    tda_b200.cache4_append(cache, x, x, x, slots)
    want = values64(*quantise64(x))
    for y in tda_b200.cache4_read(cache, slots, torch.float32):
        assert torch.equal(y.double(), want), int((y.double() != want).sum())


def test_exact_halves():
    """7 x / amax is a half exactly where amax = 7 m / 2^k: to the even code."""
    m = torch.randint(1, 1 << 20, (512, 1, 1), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    half = torch.arange(64, device=DEV) % 15 - 7.5
    half[::32] = 7.0
    half[15::15] = 0.5
    x = (half * m.float()).reshape(512, 1, 64)
    cache = tda_b200.Cache4(8, 64, 1, 64)
    slots = torch.arange(512, dtype=torch.int32, device=DEV)
    ok = x.abs() <= 7 * m.float()
    x = torch.where(ok, x, torch.zeros_like(x))
    tda_b200.cache4_append(cache, x, x, x, slots)
    want = values64(*quantise64(x))
    for y in tda_b200.cache4_read(cache, slots, torch.float32):
        assert torch.equal(y.double(), want)
