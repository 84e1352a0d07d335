"""The 4-bit paged cache: its page plan against a plain loop, codes against the
64-bit definition (equal), attention against 64 bits over the values the cache
holds.

Attention tolerance (relative 2-norm): a weight is rounded to bf16 once (2^-9
at most) and the output once; independent, so 2^-8 for bf16 and for fp16
(whose weights are bf16 as well)."""
import math

import pytest
import torch

import tda_b200
from tests.sdiff_reference import decode64, quantise64, rel, values64

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -8
DEV = "cuda"


# ------------------------------------------------------------------ plan
def plan_loop(lengths, new, table, free, head, page, rows):
    width = len(table[0])
    slots, pos, req, starts, after, dropped = [], [], [], [0], [], 0
    for r, (n, m) in enumerate(zip(lengths, new)):
        held = -(-n // page)
        want = max(0, min(-(-(n + m) // page), width) - held)
        got = min(want, max(0, len(free) - head))
        for c in range(got):
            table[r][held + c] = free[head + c]
        head += got
        cap = (held + got) * page
        for i in range(m):
            p = n + i
            pos.append(p)
            req.append(r)
            slots.append(table[r][p // page] * page + p % page if p < cap else -1)
        after.append(min(n + m, cap))
        dropped += n + m - after[-1]
        starts.append(starts[-1] + m)
    fill = lambda x: (x + [-1] * rows)[:rows]
    return fill(slots), fill(pos), fill(req), starts, after, head, dropped, table


@pytest.mark.parametrize("B,page,longest,rows_extra,short", [
    (1, 16, 1, 0, 0), (1, 64, 300, 5, 0), (7, 16, 40, 0, 0), (33, 128, 700, 11, 0), (600, 32, 90, 100, 0),
    (5000, 16, 20, 3, 0),          # more requests than one scan takes
    (40, 16, 100, 0, 60),          # the free list runs out
    (3, 16, 3000, 0, 0),           # several blocks of rows
])
def test_plan_equals_a_loop(B, page, longest, rows_extra, short):
    g = torch.Generator().manual_seed(B + page)
    lengths = torch.randint(0, longest + 1, (B,), generator=g)
    new = torch.randint(0, longest + 1, (B,), generator=g)
    new[torch.rand(B, generator=g) < 0.3] = 0
    width = -(-2 * longest // page)
    table = torch.randint(0, 1000, (B, width), generator=g)
    need = sum(-(-int(a + b) // page) - -(-int(a) // page) for a, b in zip(lengths, new))
    free = torch.randperm(max(1, need + 3 - short), generator=g)
    head = 2 if free.numel() > 2 and short == 0 else 0
    free = torch.cat([torch.full((head,), 999999), free])
    rows = int(new.sum()) + rows_extra
    want = plan_loop(lengths.tolist(), new.tolist(), table.tolist(), free.tolist(), head, page, rows)
    d = lambda t: t.to(torch.int32).to(DEV)
    wide = torch.full((B, width + 3), -5, dtype=torch.int32, device=DEV)
    wide[:, :width] = d(table)
    tab = wide[:, :width]  # rows apart by more than the width
    p = tda_b200.plan_pages(d(lengths), d(new), tab, d(free), d(torch.tensor([head])), page, rows)
    for name, w in zip(("slots", "positions", "requests", "starts", "lengths"), want):
        assert getattr(p, name).tolist() == w, name
    assert p.free_head.tolist() == [want[5]] and p.dropped.tolist() == [want[6]]
    assert tab.tolist() == want[7]
    assert (wide[:, width:] == -5).all()
    if short:
        assert want[6] > 0


def test_plan_when_the_table_is_full():
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.tensor([[3, -1], [4, 5]], dtype=torch.int32, device=DEV)
    p = tda_b200.plan_pages(i(16, 30), i(40, 9), table, i(7, 8, 9), i(0), 16, 49)
    assert p.lengths.tolist() == [32, 32] and p.dropped.tolist() == [24 + 7] and p.free_head.tolist() == [1]
    assert p.slots.tolist() == [7 * 16 + x for x in range(16)] + [-1] * 24 + [5 * 16 + 14, 5 * 16 + 15] + [-1] * 7


# ------------------------------------------------------------------ append / read
def special_rows(T, H, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, H, D, generator=g, device=DEV).to(dtype)
    x[0] = 0
    if T > 1:
        x[1] = torch.where(torch.arange(D, device=DEV) % 2 == 0, 1.0, 0.5).to(dtype)  # halves of the maximum: ties
    if T > 2:
        x[2] = (torch.randint(-14, 15, (H, D), generator=g, device=DEV).float() / 14).to(dtype)  # many near-ties
        x[2, :, 0::32] = 1.0
    if T > 3:
        x[3] *= 1e-7 if dtype != torch.float16 else 1e-4
    if T > 4 and dtype == torch.bfloat16:
        x[4] = (x[4].float() * 1e30).to(dtype)
        x[4, :, :32] = (x[4, :, :32].float() * 1e-68).to(dtype)
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("T,H", [(1, 1), (5, 3), (100, 2)])
def test_codes_equal_the_definition(dtype, D, page, T, H):
    xs = [special_rows(T, H, D, dtype, 7 * i + T) for i in range(3)]
    pages = T // page + 2
    cache = tda_b200.Cache4(pages, page, H, D)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:T].to(torch.int32).to(DEV)
    tda_b200.cache4_append(cache, *xs, slots)
    got = tda_b200.cache4_read(cache, slots, torch.float32)
    for x, y in zip(xs, got):
        assert torch.equal(y.double(), values64(*quantise64(x)))  # code x scale is exact in fp32
    # another type rounds the same value once
    for y, z in zip(got, tda_b200.cache4_read(cache, slots, torch.bfloat16)):
        assert torch.equal(y.to(torch.bfloat16), z)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_normalized_keys_strides_and_skipped_rows(dtype):
    T, H, D, page = 70, 4, 128, 32
    g = torch.Generator(device=DEV).manual_seed(3)
    fused = torch.randn(T, 3, H, D, generator=g, device=DEV).to(dtype)  # one projection's output
    k1, k2, v = fused[:, 0], fused[:, 1], fused[:, 2]
    cache = tda_b200.Cache4(4, page, H, D, normalize_keys=True)
    before = cache.data.clone()
    slots = torch.randperm(4 * page, generator=torch.Generator().manual_seed(2))[:T].to(torch.int32)
    slots[5], slots[6] = -1, 4 * page  # no slot, and one past the cache
    slots = slots.to(DEV)
    tda_b200.cache4_append(cache, k1, k2, v, slots)
    for i, (x, y) in enumerate(zip((k1, k2, v), tda_b200.cache4_read(cache, slots, torch.float32))):
        want = values64(*quantise64(x, normalize=i < 2))
        want[5:7] = 0
        # fp32 inputs and normalized scales round 1 / norm (and 7 x / amax) in fp32: a scale may land on the
        # neighbouring bf16 (2^-8 of its group), a code on the other side of a half
        assert rel(y, want) <= (2.0 ** -9 if i < 2 or dtype == torch.float32 else 0.0)
    untouched = torch.ones(4 * page, dtype=torch.bool)
    untouched[slots[(slots >= 0) & (slots < 4 * page)].long().cpu()] = False
    rest = untouched.nonzero().flatten().to(torch.int32).to(DEV)
    for y in tda_b200.cache4_read(cache, rest, torch.float32):
        assert float(y.abs().max()) == 0.0
    assert before.shape == cache.data.shape


def test_infinities_and_nan_read_back_as_nan():
    x = torch.randn(3, 1, 64, device=DEV).to(torch.bfloat16)
    x[0, 0, 5] = math.inf
    x[1, 0, 40] = math.nan
    cache = tda_b200.Cache4(1, 16, 1, 64)
    slots = torch.arange(3, dtype=torch.int32, device=DEV)
    tda_b200.cache4_append(cache, x, x, x, slots)
    for y in tda_b200.cache4_read(cache, slots, torch.float32):
        bad = torch.zeros(3, 1, 64, dtype=torch.bool, device=DEV)
        bad[0, 0, :32] = True
        bad[1, 0, 32:] = True
        assert torch.equal(torch.isnan(y), bad)


# ------------------------------------------------------------------ attention
def filled(lens, H, Hkv, D, page, dtype, seed, normalize=False, lean=0.0, poison=True, extra=2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = len(lens)
    width = max(1, -(-max(lens) // page)) + 1
    pages = sum(-(-n // page) for n in lens) + extra
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(DEV)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    cache = tda_b200.Cache4(pages, page, Hkv, D, normalize_keys=normalize)
    if poison:  # what no token was written to holds NaN scales
        cache.data.fill_(0xff)
    u = lean * torch.randn(2, Hkv, D, generator=g, device=DEV)
    at, slots_of = 0, []
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
        i = torch.arange(n, device=DEV)
        slots = (table[b, i // page] * page + i % page).to(torch.int32)
        slots_of.append(slots)
        if n:
            kv = [torch.randn(n, Hkv, D, generator=g, device=DEV) for _ in range(3)]
            tda_b200.cache4_append(cache, (kv[0] + u[0]).to(dtype), (kv[1] + u[1]).to(dtype), kv[2].to(dtype), slots)
    lift = u.repeat_interleave(H // Hkv, 1)
    q1, q2 = ((torch.randn(B, H, D, generator=g, device=DEV) + lift[i]).to(dtype) for i in range(2))
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return cache, table, lengths, slots_of, q1, q2


def expected(cache, slots_of, q1, q2, lam, **kw):
    out = []
    for b, slots in enumerate(slots_of):
        kv = tda_b200.cache4_read(cache, slots, torch.float32)
        out.append(decode64(q1[b], q2[b], *kv, lam, normalize=cache.normalize_keys, **kw))
    return torch.stack(out)


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 2), (6, 2), (10, 2), (8, 1)])
def test_softmax_form(dtype, D, page, H, Hkv):
    cache, table, lengths, slots, q1, q2 = filled(LENS, H, Hkv, D, page, dtype, H + D)
    lam = torch.linspace(-0.5, 1.5, H, device=DEV)
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, lam.reshape(1, H, 1, 1))
    want = expected(cache, slots, q1, q2, lam)
    assert out.dtype == dtype and torch.isfinite(out).all() and float(out[0].abs().max()) == 0.0
    for b in range(1, len(LENS)):
        assert rel(out[b], want[b]) <= TOL, (LENS[b], rel(out[b], want[b]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page,H,Hkv", [(64, 32, 4, 4), (128, 64, 8, 2), (128, 16, 5, 1)])
@pytest.mark.parametrize("power", [1.0, 2.0, 3.0, 1.5])
@pytest.mark.parametrize("normalize", [True, False])
def test_threshold_form(dtype, D, page, H, Hkv, power, normalize):
    cache, table, lengths, slots, q1, q2 = filled(LENS, H, Hkv, D, page, dtype, H, normalize, lean=0.6)
    beta = 0.9 if normalize else 20.0
    lam = torch.linspace(-0.2, 1.2, H, device=DEV)  # clamped to [0, 1]
    out = tda_b200.cache4_threshold_attention(q1, q2, cache, table, lengths, beta, lam.reshape(H, 1, 1), power)
    want = expected(cache, slots, q1, q2, lam, threshold=True, beta=beta, power=power)
    for b in range(1, len(LENS)):
        fits = torch.isfinite(want[b].to(dtype))  # unnormalized weights pass what fp16 holds
        assert torch.equal(torch.isfinite(out[b]), fits)
        out[b], want[b] = out[b].masked_fill(~fits, 0), want[b].masked_fill(~fits, 0)
        # a score next to the threshold: z carries the score's error of a few 2^-20 whole, weights near 0 add little
        assert rel(out[b], want[b]) <= TOL or float((out[b].double() - want[b]).abs().max()) <= 1e-5, (LENS[b], rel(out[b], want[b]))


def test_threshold_form_is_the_last_row_of_the_sequence_form():
    n, H, D = 200, 2, 64
    cache, table, lengths, slots, q1, q2 = filled([n], H, H, D, 32, torch.bfloat16, 1, True, lean=0.6)
    k1, k2, v = (t.transpose(0, 1)[None] for t in tda_b200.cache4_read(cache, slots[0], torch.float32))
    qs = [torch.zeros(1, H, n, D, device=DEV) for _ in range(2)]
    for q, x in zip(qs, (q1, q2)):
        q[0, :, -1] = x[0].float() / x[0].float().norm(dim=-1, keepdim=True)
    whole = tda_b200.differential_threshold_rela_triton(qs[0], qs[1], k1, k2, v, 1.0, torch.tensor(0.4), 2.0, False)
    one = tda_b200.cache4_threshold_attention(q1, q2, cache, table, lengths, 1.0, 0.4, 2.0)
    assert rel(one[0], whole[0, :, -1]) <= TOL


@pytest.mark.parametrize("n", [4096, 5000, 40000])
def test_long_requests_split_over_blocks(n):
    cache, table, lengths, slots, q1, q2 = filled([n, 77], 8, 2, 128, 64, torch.bfloat16, n, poison=False)
    lam = torch.full((8,), 0.4, device=DEV)
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, 0.4)
    want = expected(cache, slots, q1, q2, lam)
    assert rel(out[0], want[0]) <= TOL and rel(out[1], want[1]) <= TOL
    again = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, 0.4)
    assert torch.equal(out, again)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB, its last pages in use."""
    page, Hkv, D, H = 128, 8, 128, 8
    block = tda_b200.Cache4(1, page, 1, D).data.shape[2]
    pages = (1 << 32) // (block * Hkv) + 16
    cache = tda_b200.Cache4(pages, page, Hkv, D)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=DEV)
    n = 200
    i = torch.arange(n, device=DEV)
    slots = (table[0, i // page] * page + i % page).to(torch.int32)
    kv = [torch.randn(n, Hkv, D, device=DEV).to(torch.bfloat16) for _ in range(3)]
    tda_b200.cache4_append(cache, *kv, slots)
    for x, y in zip(kv, tda_b200.cache4_read(cache, slots, torch.float32)):
        assert torch.equal(y.double(), values64(*quantise64(x)))
    q1, q2 = (torch.randn(1, H, D, device=DEV).to(torch.bfloat16) for _ in range(2))
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, torch.tensor([n], dtype=torch.int32, device=DEV), 0.5)
    want = expected(cache, [slots], q1, q2, torch.full((H,), 0.5, device=DEV))
    assert rel(out, want) <= TOL


def test_large_scores_and_a_late_maximum():
    cache, table, lengths, slots, q1, q2 = filled([900], 4, 1, 128, 64, torch.bfloat16, 5, poison=False)
    # one late key answers the queries strongly
    kv = [t[850:851].to(torch.bfloat16) for t in tda_b200.cache4_read(cache, slots[0], torch.float32)]
    tda_b200.cache4_append(cache, (q1[0, :1] * 3)[None].to(torch.bfloat16), kv[1], kv[2], slots[0][850:851].contiguous())
    lam = torch.full((4,), 0.5, device=DEV)
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, 0.5)
    assert rel(out, expected(cache, slots, q1, q2, lam)) <= TOL
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, 0.5, scale=1.0)
    assert rel(out, expected(cache, slots, q1, q2, lam, scale=1.0)) <= 4 * TOL  # scores near 100: their fp32 error enters the weight


def test_lengths_and_pages_out_of_range_are_bounded():
    """A length past the table is cut to it; entries outside the cache are skipped."""
    cache, table, lengths, slots, q1, q2 = filled([64, 40], 2, 1, 64, 16, torch.bfloat16, 2, poison=False)
    table[0, 1], table[0, 2] = -1, 10 ** 6
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, lengths, 0.5)
    keep = torch.cat([slots[0][:16], slots[0][48:]])
    want = expected(cache, [keep, slots[1]], q1, q2, torch.full((2,), 0.5, device=DEV))
    assert rel(out, want) <= TOL
    big = torch.tensor([10 ** 9, -4], dtype=torch.int32, device=DEV)
    out = tda_b200.cache4_softmax_attention(q1, q2, cache, table, big, 0.5)
    assert rel(out[0], want[0]) <= TOL and float(out[1].abs().max()) == 0.0


def test_step_in_a_graph_and_on_another_stream():
    """plan -> append -> attention captured once and replayed with other inputs."""
    B, H, Hkv, D, page = 4, 4, 2, 64, 16
    cache = tda_b200.Cache4(64, page, Hkv, D)
    table = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(DEV)
    head = torch.zeros(1, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    ones = torch.ones(B, dtype=torch.int32, device=DEV)
    buf = [torch.zeros(B, h, D, dtype=torch.bfloat16, device=DEV) for h in (H, H, Hkv, Hkv, Hkv)]

    def step():
        p = tda_b200.plan_pages(lengths, ones, table, free, head, page, B)
        tda_b200.cache4_append(cache, *buf[2:], p.slots)
        out = tda_b200.cache4_softmax_attention(buf[0], buf[1], cache, table, p.lengths, 0.3)
        lengths.copy_(p.lengths)
        head.copy_(p.free_head)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        lengths.zero_(), head.zero_(), table.fill_(-1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lengths.zero_(), head.zero_(), table.fill_(-1), cache.data.zero_()
    g = torch.Generator(device=DEV).manual_seed(1)
    seen = [[], [], []]
    for n in range(1, 21):
        for b in buf:
            b.copy_(torch.randn(b.shape, generator=g, device=DEV))
        graph.replay()
        for s, x in zip(seen, buf[2:]):
            s.append(values64(*quantise64(x)))
        for b in range(B):
            kv = [torch.stack(s)[:, b] for s in seen]
            want = decode64(buf[0][b], buf[1][b], *kv, torch.full((H,), 0.3, device=DEV))
            assert rel(out[b], want) <= TOL, n
    assert lengths.tolist() == [20] * B and head.tolist() == [2 * B]
