"""Softmax differential attention against its 64-bit form: types, shared heads,
uneven lengths, empty rows, strides, streams, gradients.

Tolerances (relative 2-norm).  fp32: sums of at most a few thousand fp32
products, 1e-5.  bf16 / fp16: the output is rounded once (2^-9 / 2^-12 at most
an element, half that in the mean) and so are the weights before their product
with v; their errors are independent, so 2^-8 / 2^-11 holds the output.  A
gradient adds the rounding of dS and, in D, of the saved outputs: 2^-7 / 2^-10."""
import math

import pytest
import torch

import tda_b200
from tests.sdiff_reference import attention64, rel

pytestmark = pytest.mark.gpu

OUT_TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
GRAD_TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
NAMES = ("dq1", "dq2", "dk1", "dk2", "dv")


def make(B, H, Hkv, Sq, Sk, D, dtype, seed=0, bshd=False, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)

    def t(h, s):
        if bshd:
            return torch.randn(B, s, h, D, generator=g, device=dev).to(dtype).transpose(1, 2)
        return torch.randn(B, h, s, D, generator=g, device=dev).to(dtype)

    q1, q2, k1, k2, v = t(H, Sq), t(H, Sq), t(Hkv, Sk), t(Hkv, Sk), t(Hkv, Sk)
    dout = t(H, Sq)
    lam = 0.2 + 0.6 * torch.rand(1, H, 1, 1, generator=g, device=dev)
    return [q1, q2, k1, k2, v], dout, lam


def check(xs, dout, lam, causal, lengths, scale=None, backward=True):
    dtype = xs[0].dtype
    leaves = [x.detach().requires_grad_(True) for x in xs]
    lam_t = lam.detach().clone().requires_grad_(True) if isinstance(lam, torch.Tensor) else lam
    out = tda_b200.differential_softmax_attention(*leaves, lam_t, scale, causal, lengths)
    assert out.dtype == dtype and out.shape == xs[0].shape
    ref = attention64(*xs, lam, scale, causal, lengths, dout if backward else None)
    ref_out = ref[0] if backward else ref
    assert torch.isfinite(out).all()
    assert rel(out, ref_out) <= OUT_TOL[dtype], rel(out, ref_out)
    if not backward:
        return out
    grads = torch.autograd.grad(out, leaves + ([lam_t] if isinstance(lam, torch.Tensor) else []), dout)
    for n, x, g, r in zip(NAMES, xs, grads, ref[1:6]):
        assert g.dtype == x.dtype and g.shape == x.shape
        if r.norm() == 0:
            assert float(g.double().norm()) == 0.0, n
        elif (r.norm() / math.sqrt(r.numel())) > 1e-6:  # a lone key's dS is a difference of equal numbers
            assert rel(g, r) <= GRAD_TOL[dtype], (n, rel(g, r))
    if isinstance(lam, torch.Tensor):
        # dlambda sums rows of either sign: its error is held against the size of the summed terms
        dl = ref[6].sum(0)
        terms = float(dout.double().norm())
        got = grads[5].reshape(-1).double().to(dout.device)
        want = dl if lam.numel() > 1 else dl.sum().reshape(1)
        assert float((got - want).norm()) <= GRAD_TOL[dtype] * max(float(want.norm()), terms), (got, want)
    torch.cuda.synchronize()
    tda_b200.check_status()
    return out


SHAPES = [
    # B, H, Hkv, Sq, Sk, causal
    (1, 1, 1, 1, 1, True),
    (1, 2, 1, 1, 257, True),       # one query over a cached prefix
    (2, 2, 2, 127, 127, True),
    (1, 4, 2, 128, 128, True),
    (2, 3, 1, 129, 129, True),
    (1, 2, 2, 65, 300, True),      # a chunk of queries at the end of the keys
    (1, 2, 2, 300, 65, True),      # rows in front of the first key see nothing
    (2, 4, 1, 200, 333, False),
    (1, 8, 8, 513, 513, True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, D, dtype):
    B, H, Hkv, Sq, Sk, causal = shape
    xs, dout, lam = make(B, H, Hkv, Sq, Sk, D, dtype, seed=Sq + Sk + D)
    check(xs, dout, lam, causal, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 32, 256])
def test_other_head_dims(D, dtype):
    xs, dout, lam = make(2, 4, 2, 77, 77, D, dtype, seed=D)
    check(xs, dout, lam, True, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_key_lengths_hide_anything(dtype, D, causal):
    """Sequences of 0, 1, tile-edge and full length; NaN and infinities past a length stay out of results."""
    lens = [0, 1, 127, 128, 129, 200]
    xs, dout, lam = make(len(lens), 4, 2, 200, 200, D, dtype, seed=9)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for t, bad in ((xs[2], math.nan), (xs[3], math.inf), (xs[4], math.nan)):
        for b, n in enumerate(lens):
            t[b, :, n:] = bad
    out = check(xs, dout, lam, causal, lengths)
    assert float(out[0].detach().abs().max()) == 0.0
    check(xs, dout, lam, causal, lengths.long())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_strided_views_equal_copies(dtype, D):
    xs, dout, lam = make(2, 4, 2, 150, 150, D, dtype, seed=4, bshd=True)
    a = check(xs, dout, lam, True, None)
    b = tda_b200.differential_softmax_attention(*[x.contiguous() for x in xs], lam)
    assert torch.equal(a, b)
    # a slice at an address that is no multiple of 16 bytes, and a reversed axis order
    wide = torch.randn(2, 4, 150, D + 1, device="cuda").to(dtype)
    odd = wide[..., 1:]
    c = tda_b200.differential_softmax_attention(odd, *xs[1:], lam)
    d = tda_b200.differential_softmax_attention(odd.contiguous(), *xs[1:], lam)
    assert torch.equal(c, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lambda_forms(dtype):
    B, H = 2, 4
    xs, dout, _ = make(B, H, 2, 140, 140, 64, dtype, seed=5)
    g = torch.Generator(device="cuda").manual_seed(1)
    for lam in (0.0, -0.7, 1.8, torch.tensor(0.3), torch.tensor(0.3, device="cuda"),
                torch.rand(H, 1, 1, generator=g, device="cuda"),
                torch.rand(B, H, 1, 1, generator=g, device="cuda").double()):
        check(xs, dout, lam, True, None) if not (isinstance(lam, torch.Tensor) and lam.shape[0:1] == (B,) and lam.dim() == 4) \
            else _check_full_lambda(xs, dout, lam)
    half = torch.rand(1, H, 1, 1, generator=g, device="cuda").to(torch.bfloat16)
    a = tda_b200.differential_softmax_attention(*xs, half)
    b = tda_b200.differential_softmax_attention(*xs, half.float())
    assert torch.equal(a, b)


def _check_full_lambda(xs, dout, lam):
    dtype = xs[0].dtype
    l = lam.clone().requires_grad_(True)
    out = tda_b200.differential_softmax_attention(*xs, l)
    ref = attention64(*xs, lam, dout=dout)
    assert rel(out, ref[0]) <= OUT_TOL[dtype]
    (dl,) = torch.autograd.grad(out, [l], dout)
    assert dl.shape == lam.shape and dl.dtype == lam.dtype
    terms = float(dout.double().norm())
    assert float((dl.reshape(-1).double() - ref[6].reshape(-1)).norm()) <= GRAD_TOL[dtype] * terms


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_large_scores(dtype):
    """Scores in the hundreds: weights that are 0 or 1, rows whose maximum moves from tile to tile."""
    xs, dout, lam = make(1, 2, 2, 400, 400, 64, dtype, seed=6)
    ramp = torch.linspace(0.2, 6.0, 400, device="cuda")[:, None].to(dtype)
    xs[2], xs[3] = xs[2] * ramp, xs[3] * ramp
    out = tda_b200.differential_softmax_attention(*xs, lam, 1.0)
    ref = attention64(*xs, lam, 1.0)
    assert rel(out, ref) <= 4 * OUT_TOL[dtype]  # a weight's relative error is the score's absolute one: fp32 of some hundred


def test_a_score_outside_the_range_of_its_neighbours():
    """A key far above all before it: the running maximum jumps by more than any lazy margin."""
    xs, dout, lam = make(1, 1, 1, 300, 300, 128, torch.bfloat16, seed=8)
    xs[0][:, :, 290:] *= 4
    xs[2][:, :, 280] = xs[0][:, :, 295] * 2
    check(xs, dout, lam, True, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_gradient_against_differences(dtype, D):
    """d/de of sum(out dout) along a random direction, by differences of the 64-bit form at the kernel's gradient point;
    the step's truncation, e^2 times a third derivative near 1, is below 1e-6 at e = 1e-3."""
    xs, dout, lam = make(1, 2, 1, 96, 96, D, dtype, seed=11)
    leaves = [x.detach().requires_grad_(True) for x in xs]
    l = lam.clone().requires_grad_(True)
    out = tda_b200.differential_softmax_attention(*leaves, l)
    grads = torch.autograd.grad(out, leaves + [l], dout)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for k in range(6):
        base = [x.double() for x in xs] + [lam.double()]
        d = torch.randn(base[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        vals = []
        for e in (1e-3, -1e-3):
            moved = list(base)
            moved[k] = moved[k] + e * d
            vals.append(float((attention64(*moved[:5], moved[5]) * dout.double()).sum()))
        slope = (vals[0] - vals[1]) / 2e-3
        got = float((grads[k].double() * d).sum())
        # a random direction turns a relative error of the gradient into that share of |gradient| (times a normal variate)
        assert abs(got - slope) <= 4 * GRAD_TOL[dtype] * float(grads[k].double().norm()) + 1e-5, (k, got, slope)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_bits_every_time_and_on_another_stream(dtype):
    xs, dout, lam = make(2, 4, 1, 260, 260, 128, dtype, seed=12)
    leaves = [x.detach().requires_grad_(True) for x in xs]

    def step():
        out = tda_b200.differential_softmax_attention(*leaves, lam)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    a = step()
    b = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = step()
    torch.cuda.current_stream().wait_stream(s)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_mixed_and_wide_types():
    xs, dout, lam = make(1, 2, 2, 70, 70, 64, torch.float64, seed=13)
    out = tda_b200.differential_softmax_attention(*xs, lam)
    assert out.dtype == torch.float64 and rel(out, attention64(*xs, lam)) <= 1e-5
    mixed = [xs[0].to(torch.bfloat16), xs[1].to(torch.bfloat16)] + [x.float() for x in xs[2:]]
    out = tda_b200.differential_softmax_attention(*mixed, lam)
    assert out.dtype == torch.bfloat16 and rel(out, attention64(*mixed, lam)) <= OUT_TOL[torch.bfloat16]


def test_empty_inputs():
    z = torch.zeros(2, 4, 0, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(2, 4, 5, 64, device="cuda", dtype=torch.bfloat16)
    assert tda_b200.differential_softmax_attention(z, z, k, k, k, 0.5).shape == z.shape
    q = torch.ones(2, 4, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = tda_b200.differential_softmax_attention(q, q, z, z, z, 0.5)
    assert float(out.detach().abs().max()) == 0.0
    (g,) = torch.autograd.grad(out, [q], torch.ones_like(out))
    assert float(g.abs().max()) == 0.0


def test_cuda_graph_and_compile():
    xs, dout, lam = make(1, 2, 2, 200, 200, 64, torch.bfloat16, seed=14)
    eager = tda_b200.differential_softmax_attention(*xs, lam)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tda_b200.differential_softmax_attention(*xs, lam)
    captured.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, captured)
    leaves = [x.detach().requires_grad_(True) for x in xs]
    l = lam.clone().requires_grad_(True)
    fn = torch.compile(lambda *a: tda_b200.differential_softmax_attention(*a), fullgraph=True, backend="aot_eager")
    out = fn(*leaves, l)
    assert torch.equal(out, eager)
    g1 = torch.autograd.grad(out, leaves + [l], dout)
    g2 = torch.autograd.grad(tda_b200.differential_softmax_attention(*leaves, l), leaves + [l], dout)
    for x, y in zip(g1, g2):
        assert torch.equal(x, y)


@pytest.mark.parametrize("shape", [
    # B, H, Hkv, S, D, dtype: heads that make several groups of tiles, of a prime number of heads, of one head
    (3, 40, 8, 1025, 16, torch.float32),
    (20, 6, 3, 1300, 64, torch.bfloat16),
    (1, 37, 37, 1999, 64, torch.float16),
    (2, 5, 5, 4300, 64, torch.bfloat16),
])
def test_causal_tiles_of_many_heads(shape):
    """Every tile of every head is computed once whatever the number of heads that run side by side."""
    B, H, Hkv, S, D, dtype = shape
    xs, dout, lam = make(B, H, Hkv, S, S, D, dtype, seed=S)
    check(xs, dout, lam, True, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Sk,causal", [(700, 700, True), (300, 700, True), (700, 300, True), (520, 640, False)])
def test_weights_around_512_keys(Sq, Sk, causal, dtype):
    """dv where some query tiles see 512 keys or fewer, and lengths on either side of that."""
    lens = torch.tensor([n for n in (511, 512, 513, Sk) if n <= Sk], dtype=torch.int32, device="cuda")
    xs, dout, lam = make(len(lens), 4, 2, Sq, Sk, 128, dtype, seed=Sq)
    check(xs, dout, lam, causal, lens)
