"""Cases for the operators around differential attention: softmax differential
attention (forward and training step), the page plan of a serving step, the
4-bit cache (append, read) and one-token attention over it.

``run`` computes the plain form (elementary torch operations in fp32) where
``own`` is false and calls ``tda_b200`` where it is true.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 32  # elements along the head dimension that share one scale of the 4-bit cache
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK_ELEMS = 1 << 28  # score elements the plain form holds at a time


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one short prompt on 8 small heads: the smallest call of this package's tests; launch latency counts
        dict(name="prompt_short", op="forward", dtype="bf16", b=1, hq=8, hkv=8, sq=128, sk=128, d=64, causal=True,
             ragged=False, lam="scalar", bshd=False),
        # long-context prefill, the benchmark's longest sequence
        dict(name="prompt_long", op="forward", dtype="bf16", b=1, hq=16, hkv=16, sq=32768, sk=32768, d=128, causal=True,
             ragged=False, lam="head", bshd=False),
        # a training layer with shared key / value heads at the benchmark's (4, 32, 4096, 128)
        dict(name="train_grouped", op="train", dtype="bf16", b=4, hq=32, hkv=8, sq=4096, sk=4096, d=128, causal=True,
             ragged=False, lam="head", bshd=True),
        # a padded fp16 batch of odd length with per-sequence key lengths (one of them empty), not causal
        dict(name="train_padded", op="train", dtype="fp16", b=6, hq=16, hkv=16, sq=1999, sk=1999, d=64, causal=False,
             ragged=True, lam="head", bshd=False),
        # fp32 as a debugging run uses it
        dict(name="train_fp32", op="train", dtype="fp32", b=2, hq=16, hkv=8, sq=1024, sk=1024, d=64, causal=True,
             ragged=False, lam="head", bshd=False),
        # book-keeping of one decode step of 256 requests
        dict(name="plan_step", op="plan", b=256, page=64, longest=8192, new="one"),
        # book-keeping of a step that admits many prompts
        dict(name="plan_prompts", op="plan", b=512, page=16, longest=4096, new="many"),
        # cache write of one decode step: 256 tokens of 8 kv heads, and their read-back
        dict(name="append_step", op="append", dtype="bf16", tokens=256, hkv=8, d=128, page=64, normalize=True),
        # cache write and read-back of packed prompts
        dict(name="append_prompts", op="append", dtype="bf16", tokens=32768, hkv=8, d=128, page=64, normalize=False),
        # one request at a long context, 4 query heads to a kv head
        dict(name="decode_one", op="decode", map="softmax", dtype="bf16", b=1, hq=32, hkv=8, d=128, page=64,
             longest=32768, even=True, lam="head"),
        # a serving batch of uneven lengths
        dict(name="decode_batch", op="decode", map="softmax", dtype="bf16", b=128, hq=32, hkv=8, d=128, page=64,
             longest=16384, even=False, lam="head"),
        # the threshold form over the same kind of batch, heads not shared
        dict(name="decode_threshold", op="decode", map="threshold", dtype="bf16", b=32, hq=16, hkv=16, d=128, page=16,
             longest=8192, even=False, lam="scalar"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _draw(rng)
    if case["op"] in ("forward", "train", "decode"):
        # no dearer than the largest listed case of its kind
        kind = lambda c: (c["op"], c.get("dtype") == "fp32")
        top = max(work(c)["flops"] + work(c)["bytes"] for c in listed() if kind(c) == kind(case))
        while work(case)["flops"] + work(case)["bytes"] > top:
            for k in ("sq", "sk", "longest"):
                if k in case:
                    case[k] = max(1, case[k] * 3 // 4)
            if "sq" in case:
                case["sq"] = min(case["sq"], case["sk"])
    return case


def _draw(rng):
    op = rng.choice(["forward", "train", "train", "plan", "append", "decode", "decode", "decode"])
    if op in ("forward", "train"):
        d = rng.choice([64, 128, 128])
        dtype = rng.choice(["bf16", "bf16", "fp16"] + (["fp32"] if op == "train" else []))
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4])
        b = rng.choice([1, 2, 3, 4])
        top = 1024 if dtype == "fp32" else 4096 if op == "train" else 16384
        sk = _log_int(rng, 1, top)
        shape = rng.choice(["square", "square", "chunk"])
        sq = sk if shape == "square" else rng.randint(1, sk)
        ragged = rng.random() < 0.4
        lam = rng.choice(["scalar", "head"])
        if op == "train":  # a lone lambda's gradient is one sum of terms of either sign, which cancel: a layer has several heads
            lam, hkv, hq = "head", max(hkv, 8 * hkv // hq), max(hq, 8)
        return dict(op=op, dtype=dtype, b=b, hq=hq, hkv=hkv, sq=sq, sk=sk, d=d, causal=rng.random() < 0.7,
                    ragged=ragged, lam=lam, bshd=rng.random() < 0.5)
    if op == "plan":
        return dict(op=op, b=_log_int(rng, 1, 512), page=rng.choice([16, 32, 64, 128]), longest=_log_int(rng, 1, 4096),
                    new=rng.choice(["one", "many"]))
    if op == "append":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), tokens=_log_int(rng, 1, 32768), hkv=rng.choice([1, 2, 4, 8]),
                    d=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), normalize=rng.random() < 0.5)
    hkv = rng.choice([1, 2, 4, 8])
    return dict(op=op, map=rng.choice(["softmax", "threshold"]), dtype=rng.choice(["bf16", "fp16"]),
                b=_log_int(rng, 1, 128), hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv, d=rng.choice([64, 128]),
                page=rng.choice([16, 32, 64, 128]), longest=_log_int(rng, 1, 16384), even=rng.random() < 0.3,
                lam=rng.choice(["scalar", "head"]))


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _lambda(case, g):
    shape = (1, case["hq"], 1, 1) if case["lam"] == "head" else ()
    return (0.2 + 0.6 * torch.rand(shape, generator=g, device=DEV)).to(DTYPES[case["dtype"]])  # a parameter in the model's type


def _attention_inputs(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    b, hq, hkv, sq, sk, d = (case[k] for k in ("b", "hq", "hkv", "sq", "sk", "d"))

    def make(h, s):
        if case["bshd"]:  # a projection's output, heads brought forward as a view
            return torch.randn((b, s, h, d), generator=g, device=DEV).to(dt).transpose(1, 2)
        return torch.randn((b, h, s, d), generator=g, device=DEV).to(dt)

    x = dict(q1=make(hq, sq), q2=make(hq, sq), k1=make(hkv, sk), k2=make(hkv, sk), v=make(hkv, sk))
    x["lam"] = _lambda(case, g)
    if case["ragged"]:
        n = torch.randint(1, sk + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        n[-1] = 0 if b > 1 else sk
        x["lengths"] = n
    else:
        x["lengths"] = None
    if case["op"] == "train":
        x["dout"] = make(hq, sq)
    return x


def _plan_rows(case):
    """Rows of the step's token buffers, which the program allocates once."""
    return case["b"] if case["new"] == "one" else (case["b"] // 2 + 1) * case["longest"]


def _plan_inputs(case, seed):
    g = _gen(seed)
    b, page, longest = case["b"], case["page"], case["longest"]
    have = torch.randint(0, longest + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    if case["new"] == "one":
        new = torch.ones((b,), device=DEV, dtype=torch.int32)
        most = 1
    else:  # half of the requests are new prompts, the rest decode one token or wait
        new = torch.randint(0, longest + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        idle = torch.rand((b,), generator=g, device=DEV)
        have = torch.where(idle < 0.5, torch.zeros_like(have), have)
        new = torch.where(idle < 0.5, new, (idle < 0.9).to(torch.int32))
        most = longest
    width = (longest + most + page - 1) // page
    pages = b * width
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    table = order.view(b, width).clone()
    held = (have + page - 1) // page
    table[torch.arange(width, device=DEV)[None, :] >= held[:, None]] = -1
    free = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    return dict(lengths=have, new=new, table=table, free=free,
                head=torch.zeros((1,), device=DEV, dtype=torch.int32), page=page,
                tokens=_plan_rows(case))


def _append_inputs(case, seed):
    g = _gen(seed)
    t, hkv, d, page = case["tokens"], case["hkv"], case["d"], case["page"]
    dt = DTYPES[case["dtype"]]
    k1, k2, v = (torch.randn((t, hkv, d), generator=g, device=DEV).to(dt) for _ in range(3))
    pages = (t + page - 1) // page + 1
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:t].to(torch.int32)
    if t > 8:  # rows of the packed batch that hold no token
        slots[t // 2] = -1
    return dict(k1=k1, k2=k2, v=v, slots=slots, pages=pages)


def _decode_lengths(case, seed):
    b, longest = case["b"], case["longest"]
    if case["even"]:
        return [longest] * b
    g = torch.Generator().manual_seed((int(seed) + 77) & 0x7FFFFFFF)
    n = torch.randint(1, longest + 1, (b,), generator=g).tolist()
    if b > 2:
        n[0], n[1] = longest, 0  # one request at the full length, one that holds nothing yet
    return n


def _decode_tokens(case, seed, request, n):
    """The keys and values of one request's n cached tokens.  Keys lean on a
    direction of their head, as a trained model's do: so the threshold form
    keeps some of them."""
    g = _gen(int(seed) * 1009 + 17 * request + 5)
    dt = DTYPES[case["dtype"]]
    kv = [torch.randn((n, case["hkv"], case["d"]), generator=g, device=DEV) for _ in range(3)]
    lean = _lean(case, seed)
    return [(t + lean[i] if i < 2 else t).to(dt) for i, t in enumerate(kv)]


def _lean(case, seed):
    g = _gen(int(seed) * 31 + 3)
    return 0.6 * torch.randn((2, case["hkv"], case["d"]), generator=g, device=DEV)


def _decode_inputs(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    b, hq, d, page = case["b"], case["hq"], case["d"], case["page"]
    lengths = _decode_lengths(case, seed)
    lean = _lean(case, seed).repeat_interleave(hq // case["hkv"], dim=1)
    q1, q2 = ((torch.randn((b, hq, d), generator=g, device=DEV) + lean[i]).to(dt) for i in range(2))
    lam = _lambda(case, g)
    lam = lam if case["lam"] == "scalar" else lam.reshape(1, hq, 1, 1)
    held = [(n + page - 1) // page for n in lengths]
    width = max(1, (case["longest"] + page - 1) // page)
    pages = sum(held) + 1
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int32)
    table = torch.full((b, width), -1, device=DEV, dtype=torch.int32)
    at = 0
    for r, m in enumerate(held):
        table[r, :m] = order[at:at + m]
        at += m
    return dict(q1=q1, q2=q2, lam=lam, table=table, pages=pages, host_lengths=lengths,
                lengths=torch.tensor(lengths, device=DEV, dtype=torch.int32))


def prepare(case, seed):
    op = case["op"]
    if op in ("forward", "train"):
        x = _attention_inputs(case, seed)
        if own and op == "train":
            for k in ("q1", "q2", "k1", "k2", "v", "lam"):
                x[k].requires_grad_(True)
        return dict(case=case, x=x)
    if op == "plan":
        return dict(case=case, x=_plan_inputs(case, seed))
    if op == "append":
        x = _append_inputs(case, seed)
        if own:
            import tda_b200
            x["cache"] = tda_b200.Cache4(x["pages"], case["page"], case["hkv"], case["d"], DEV,
                                         normalize_keys=case["normalize"])
        else:
            shape = (3, x["pages"] * case["page"], case["hkv"], case["d"])
            x["codes"] = torch.zeros(shape, device=DEV, dtype=torch.int8)
            x["scales"] = torch.zeros(shape[:3] + (case["d"] // GROUP,), device=DEV, dtype=torch.bfloat16)
        return dict(case=case, x=x)
    x = _decode_inputs(case, seed)
    page, norm = case["page"], case["map"] == "threshold"
    if own:
        import tda_b200
        x["cache"] = tda_b200.Cache4(x["pages"], page, case["hkv"], case["d"], DEV, normalize_keys=norm)
        for r, n in enumerate(x["host_lengths"]):
            if n:
                pos = torch.arange(n, device=DEV)
                slots = (x["table"][r][pos // page] * page + pos % page).to(torch.int32)
                tda_b200.cache4_append(x["cache"], *_decode_tokens(case, seed, r, n), slots)
    else:
        x["held"] = []
        for r, n in enumerate(x["host_lengths"]):
            kv = _decode_tokens(case, seed, r, n)
            x["held"].append([_quantise(t, norm and i < 2) for i, t in enumerate(kv)])
    return dict(case=case, x=x)


# ------------------------------------------------------------------ the plain forms
def _quantise(x, normalize):
    """Codes (int8, -7..7) and bf16 scales of groups of 32 along the last dimension."""
    xf = x.float()
    gr = xf.reshape(x.shape[:-1] + (x.shape[-1] // GROUP, GROUP))
    top = gr.abs().amax(-1)
    code = torch.where(top[..., None] > 0, torch.round(gr * 7.0 / top[..., None]), torch.zeros_like(gr))
    s = top / 7.0
    if normalize:
        s = s * (1.0 / torch.sqrt((xf * xf).sum(-1)).clamp_min(1e-12))[..., None]
    return code.to(torch.int8).reshape(x.shape), s.to(torch.bfloat16)


def _values(code, scale):
    gr = code.float().reshape(code.shape[:-1] + (code.shape[-1] // GROUP, GROUP))
    return (gr * scale.float()[..., None]).reshape(code.shape)


def _visible(case, x, rows):
    """Which keys each query row of each sequence sees: (b or 1, rows, sk)."""
    sk = case["sk"]
    j = torch.arange(sk, device=DEV)
    keep = torch.ones((1, rows.numel(), sk), device=DEV, dtype=torch.bool)
    if case["causal"]:
        keep = keep & (j[None, None, :] <= rows[None, :, None] + (sk - case["sq"]))
    if x["lengths"] is not None:
        keep = keep & (j[None, None, :] < x["lengths"].long()[:, None, None])
    return keep


def _heads(t, group):
    """(b, h, s, d) as fp32 (b * h * group, s, d), each kv head repeated for its query heads."""
    t = t.float()
    if group > 1:
        t = t.repeat_interleave(group, dim=1)
    return t.reshape(-1, t.shape[2], t.shape[3])


def _softmax_rows(s, keep):
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z == 0, torch.ones_like(z), z)


def _plain_attention(case, x):
    hq, sq, sk, d, b = case["hq"], case["sq"], case["sk"], case["d"], case["b"]
    group = hq // case["hkv"]
    scale = 1.0 / math.sqrt(d)
    dt = DTYPES[case["dtype"]]
    q1, q2 = _heads(x["q1"].detach(), 1), _heads(x["q2"].detach(), 1)
    k1, k2, v = (_heads(x[n].detach(), group) for n in ("k1", "k2", "v"))
    if x["lengths"] is not None:
        live = (torch.arange(sk, device=DEV)[None, :] < x["lengths"].long()[:, None]).repeat_interleave(hq, 0)[..., None]
        k1, k2, v = (torch.where(live, t, torch.zeros_like(t)) for t in (k1, k2, v))
    lam = x["lam"].detach().float().expand(b, hq, 1, 1).reshape(b * hq, 1, 1)
    n = b * hq
    train = case["op"] == "train"
    out = torch.empty((n, sq, d), device=DEV)
    row_block = max(1, min(sq, BLOCK_ELEMS // sk))
    head_block = max(1, BLOCK_ELEMS // (row_block * sk))
    if train:
        do = _heads(x["dout"], 1)
        dq1, dq2 = torch.empty_like(q1), torch.empty_like(q2)
        dk1, dk2, dv = torch.zeros_like(k1), torch.zeros_like(k2), torch.zeros_like(v)
        dlam = torch.zeros((n,), device=DEV)
    for h0 in range(0, n, head_block):
        h = slice(h0, min(n, h0 + head_block))
        for r0 in range(0, sq, row_block):
            r = slice(r0, min(sq, r0 + row_block))
            keep = _visible(case, x, torch.arange(r.start, r.stop, device=DEV))
            if keep.shape[0] > 1:
                keep = keep.repeat_interleave(hq, 0)[h]
            p1 = _softmax_rows(torch.matmul(q1[h, r], k1[h].transpose(1, 2)) * scale, keep)
            p2 = _softmax_rows(torch.matmul(q2[h, r], k2[h].transpose(1, 2)) * scale, keep)
            pc = p1 - lam[h] * p2
            out[h, r] = torch.matmul(pc, v[h])
            if train:
                g = do[h, r]
                dp = torch.matmul(g, v[h].transpose(1, 2))
                dv[h] += torch.matmul(pc.transpose(1, 2), g)
                d1, d2 = (p1 * dp).sum(-1, keepdim=True), (p2 * dp).sum(-1, keepdim=True)
                dlam[h] -= d2.sum((1, 2))
                ds1 = p1 * (dp - d1) * scale
                ds2 = -lam[h] * p2 * (dp - d2) * scale
                dq1[h, r], dq2[h, r] = torch.matmul(ds1, k1[h]), torch.matmul(ds2, k2[h])
                dk1[h] += torch.matmul(ds1.transpose(1, 2), q1[h, r])
                dk2[h] += torch.matmul(ds2.transpose(1, 2), q2[h, r])
    out = out.reshape(b, hq, sq, d).to(dt)
    if not train:
        return out
    shared = [t.reshape(b, case["hkv"], group, sk, d).sum(2).to(dt) for t in (dk1, dk2, dv)]
    dlam = dlam.reshape(b, hq).sum(0).reshape(1, hq, 1, 1) if case["lam"] == "head" else dlam.sum()
    return [out, dq1.reshape(b, hq, sq, d).to(dt), dq2.reshape(b, hq, sq, d).to(dt)] + shared + [dlam.to(dt)]


def _plain_plan(x):
    page, table = x["page"], x["table"]
    have, new = x["lengths"].long(), x["new"].long()
    width = table.shape[1]
    held = (have + page - 1) // page
    want = ((have + new + page - 1) // page).clamp(max=width) - held
    first = torch.cumsum(want, 0) - want
    left = x["free"].numel() - x["head"].long()
    got = torch.minimum(want, (left - first).clamp(min=0))
    column = torch.arange(width, device=DEV)[None, :]
    fresh = (column >= held[:, None]) & (column < (held + got)[:, None])
    take = (x["head"].long() + first[:, None] + column - held[:, None]).clamp(0, x["free"].numel() - 1)
    table = torch.where(fresh, x["free"][take], table)
    after = torch.minimum(have + new, (held + got) * page)
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros((1,), device=DEV, dtype=torch.long), ends])
    i = torch.arange(x["tokens"], device=DEV)
    live = i < ends[-1]
    req = torch.searchsorted(ends, i, right=True).clamp(max=have.numel() - 1)
    pos = have[req] + i - starts[req]
    entry = table[req, (pos // page).clamp(0, width - 1)].long()
    slot = torch.where(live & (pos < after[req]), entry * page + pos % page, torch.full_like(pos, -1))
    none = torch.full_like(pos, -1)
    to = lambda t: t.to(torch.int32)
    return dict(slots=to(slot), positions=to(torch.where(live, pos, none)), requests=to(torch.where(live, req, none)),
                starts=to(starts), lengths=to(after), table=table, free_head=to(x["head"].long() + got.sum()),
                dropped=to((have + new - after).sum().reshape(1)))


def _plain_append(case, x):
    live = x["slots"] >= 0
    to = x["slots"].long()
    for i, t in enumerate((x["k1"], x["k2"], x["v"])):
        code, scale = _quantise(t, case["normalize"] and i < 2)
        x["codes"][i][to[live]] = code[live]
        x["scales"][i][to[live]] = scale[live]
    at = to.clamp(min=0)
    dt = DTYPES[case["dtype"]]
    return [torch.where(live[:, None, None], _values(x["codes"][i][at], x["scales"][i][at]), 0.0).to(dt) for i in range(3)]


BETA, POWER = 1.0, 2.0


def _plain_decode(case, x):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    group = hq // hkv
    lam = x["lam"].float().expand(1, hq, 1, 1).reshape(hq, 1)
    out = []
    for r, n in enumerate(x["host_lengths"]):
        if n == 0:
            out.append(torch.zeros((hq, d), device=DEV))
            continue
        k1, k2, v = (_values(*t).transpose(0, 1) for t in x["held"][r])  # (hkv, n, d)
        maps = []
        for q, k in ((x["q1"], k1), (x["q2"], k2)):
            q = q[r].float()
            if case["map"] == "threshold":
                q = q * (1.0 / torch.sqrt((q * q).sum(-1, keepdim=True)).clamp_min(1e-12))
            s = torch.matmul(q.reshape(hkv, group, d), k.transpose(1, 2))
            if case["map"] == "threshold":
                tau = BETA * math.sqrt(2.0 * math.log(n) / d)
                p = (s - tau).clamp_min(0.0) ** POWER
            else:
                s = s * (1.0 / math.sqrt(d))
                e = torch.exp(s - s.amax(-1, keepdim=True))
                p = e / e.sum(-1, keepdim=True)
            maps.append(p)
        w = lam.reshape(hkv, group, 1)
        w = w.clamp(0.0, 1.0) if case["map"] == "threshold" else w
        out.append(torch.matmul(maps[0] - w * maps[1], v).reshape(hq, d))
    return torch.stack(out).to(DTYPES[case["dtype"]])


# ------------------------------------------------------------------ one pass
def run(state):
    case, x = state["case"], state["x"]
    op = case["op"]
    if not own:
        if op in ("forward", "train"):
            return _plain_attention(case, x)
        if op == "plan":
            return _plain_plan(x)
        return _plain_append(case, x) if op == "append" else _plain_decode(case, x)
    import tda_b200
    if op in ("forward", "train"):
        out = tda_b200.differential_softmax_attention(x["q1"], x["q2"], x["k1"], x["k2"], x["v"], x["lam"],
                                                      causal=case["causal"], key_lengths=x["lengths"])
        if op == "forward":
            return out
        leaves = [x[k] for k in ("q1", "q2", "k1", "k2", "v", "lam")]
        return [out.detach()] + list(torch.autograd.grad(out, leaves, x["dout"]))
    if op == "plan":
        p = tda_b200.plan_pages(x["lengths"], x["new"], x["table"], x["free"], x["head"], x["page"], x["tokens"])
        return dict(slots=p.slots, positions=p.positions, requests=p.requests, starts=p.starts, lengths=p.lengths,
                    table=x["table"], free_head=p.free_head, dropped=p.dropped)
    if op == "append":
        tda_b200.cache4_append(x["cache"], x["k1"], x["k2"], x["v"], x["slots"])
        return list(tda_b200.cache4_read(x["cache"], x["slots"], DTYPES[case["dtype"]]))
    if case["map"] == "softmax":
        return tda_b200.cache4_softmax_attention(x["q1"], x["q2"], x["cache"], x["table"], x["lengths"], x["lam"])
    return tda_b200.cache4_threshold_attention(x["q1"], x["q2"], x["cache"], x["table"], x["lengths"], BETA, x["lam"],
                                               POWER)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case, lengths):
    """Visible (query, key) pairs of one head, summed over the batch."""
    sq, sk = case["sq"], case["sk"]
    total = 0
    for n in lengths:
        if not case["causal"]:
            total += sq * n
            continue
        first = sk - sq + 1  # keys that row 0 sees (may be below 1)
        lo, hi = max(0, min(n, first)), max(0, min(n, sk))
        # rows see first, first + 1, ..., sk keys, cut at n
        ramp = hi - lo + 1 if hi >= lo else 0
        ramp = min(ramp, sq)
        total += ramp * (lo + hi) // 2 + (sq - ramp) * n
    return total


def work(case):
    op = case["op"]
    if op in ("forward", "train"):
        e = BYTES[case["dtype"]]
        lengths = [case["sk"]] * case["b"]
        if case["ragged"]:  # lengths are uniform on 1..sk, one sequence is empty
            lengths = [(case["sk"] + 1) // 2] * (case["b"] - 1) + [0] if case["b"] > 1 else lengths
        q = case["b"] * case["hq"] * case["sq"] * case["d"] * e
        kv = case["hkv"] * sum(lengths) * case["d"] * e
        product = 2 * _pairs(case, lengths) * case["hq"] * case["d"]
        if op == "forward":  # two score products and one with the values
            return dict(bytes=3 * q + 3 * kv, flops=3 * product)
        # backward: dP, dV, two each of dQ and dK; q, dout and out against dq, and k, v against their gradients
        return dict(bytes=6 * q + 6 * kv, flops=9 * product)
    if op == "plan":
        t = _plan_rows(case)
        return dict(bytes=case["b"] * 4 * 5 + t * 4 * 3 + 2 * 4 * (t // 2 // case["page"] + 1), flops=t)
    if op == "append":
        n = case["tokens"] * case["hkv"] * case["d"] * 3
        return dict(bytes=2 * n + 2 * (n // 2 + n // GROUP * 2) + 2 * n + 4 * case["tokens"], flops=2 * n)
    mean = case["longest"] if case["even"] else (case["longest"] + 1) / 2
    tokens = int(case["b"] * mean)
    d, hkv, hq = case["d"], case["hkv"], case["hq"]
    return dict(bytes=tokens * hkv * 3 * (d // 2 + d // GROUP * 2) + 3 * case["b"] * hq * d * 2,
                flops=3 * 2 * tokens * hq * d)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(case, seed):
    x = _attention_inputs(case, seed)
    b, hq, hkv, sq, sk, d = (case[k] for k in ("b", "hq", "hkv", "sq", "sk", "d"))
    train = case["op"] == "train"
    out = torch.empty((b, hq, sq, d), dtype=torch.float64, device=DEV)
    grads = {}
    if train:
        grads = {k: torch.zeros(x[k].shape, dtype=torch.float64, device=DEV) for k in ("q1", "q2", "k1", "k2", "v")}
        dl = torch.zeros((hq,), dtype=torch.float64, device=DEV)
    lam_all = x["lam"].double().reshape(-1).expand(hq) if case["lam"] == "scalar" else x["lam"].double().reshape(hq)
    step = max(1, min(sq, (1 << 27) // max(sk, 1)))
    for i in range(b):
        n = sk if x["lengths"] is None else int(x["lengths"][i].item())
        for h in range(hq):
            kv = h // (hq // hkv)
            if n == 0:
                out[i, h] = 0.0
                continue
            k1, k2, v = (x[t][i, kv, :n].double() for t in ("k1", "k2", "v"))
            lam = lam_all[h].clone()
            for r0 in range(0, sq, step):
                r1 = min(sq, r0 + step)
                last = torch.arange(r0, r1, device=DEV) + (sk - sq) if case["causal"] else torch.full((r1 - r0,), sk, device=DEV)
                hidden = torch.arange(n, device=DEV)[None, :] > last[:, None]
                empty = hidden.all(1)
                leaves = [x["q1"][i, h, r0:r1].double(), x["q2"][i, h, r0:r1].double(), k1, k2, v, lam]
                if train:
                    leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
                a1, a2, b1, b2, w, l = leaves
                maps = []
                for a, kk in ((a1, b1), (a2, b2)):
                    s = ((a @ kk.T) / d ** 0.5).masked_fill(hidden, -math.inf).masked_fill(empty[:, None], 0.0)
                    maps.append(torch.softmax(s, -1).masked_fill(empty[:, None], 0.0))
                o = maps[0] @ w - l * (maps[1] @ w)
                out[i, h, r0:r1] = o.detach()
                if train:
                    gr = torch.autograd.grad(o, leaves, x["dout"][i, h, r0:r1].double())
                    grads["q1"][i, h, r0:r1], grads["q2"][i, h, r0:r1] = gr[0], gr[1]
                    grads["k1"][i, kv, :n] += gr[2]
                    grads["k2"][i, kv, :n] += gr[3]
                    grads["v"][i, kv, :n] += gr[4]
                    dl[h] += gr[5]
    if not train:
        return out
    dl = dl.reshape(1, hq, 1, 1) if case["lam"] == "head" else dl.sum()
    return [out] + [grads[k] for k in ("q1", "q2", "k1", "k2", "v")] + [dl]


def _exact_values(t, normalize):
    """What the 4-bit cache holds for rows t, in 64 bits: code times the bf16 scale."""
    w = t.double()
    parts = []
    for part in w.split(GROUP, dim=-1):
        top = part.abs().max(dim=-1, keepdim=True).values
        code = torch.round(part * 7.0 / top.masked_fill(top == 0, 1.0))
        step = top / 7.0
        if normalize:
            step = step / w.norm(dim=-1, keepdim=True).clamp_min(1e-12)
        parts.append(code * step.float().to(torch.bfloat16).double())
    return torch.cat(parts, dim=-1)


def _exact_decode(case, seed):
    x = _decode_inputs(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    thr = case["map"] == "threshold"
    lam = x["lam"].double().reshape(-1).expand(hq) if case["lam"] == "scalar" else x["lam"].double().reshape(hq)
    out = torch.zeros((case["b"], hq, d), dtype=torch.float64, device=DEV)
    for r, n in enumerate(x["host_lengths"]):
        if n == 0:
            continue
        kv = _decode_tokens(case, seed, r, n)
        k1, k2, v = (_exact_values(t, thr and i < 2) for i, t in enumerate(kv))
        for h in range(hq):
            c = h // (hq // hkv)
            p = []
            for q, k in ((x["q1"], k1), (x["q2"], k2)):
                a = q[r, h].double()
                if thr:
                    a = a / a.norm().clamp_min(1e-12)
                    p.append(torch.relu(k[:, c] @ a - BETA * math.sqrt(2 * math.log(n) / d)) ** POWER)
                else:
                    p.append(torch.softmax((k[:, c] @ a) / d ** 0.5, 0))
            l = lam[h].clamp(0, 1) if thr else lam[h]
            out[r, h] = p[0] @ v[:, c] - l * (p[1] @ v[:, c])
    return out


def exact(case, seed):
    op = case["op"]
    if op in ("forward", "train"):
        return _exact_attention(case, seed)
    if op == "plan":
        return None
    if op == "append":
        x = _append_inputs(case, seed)
        dead = (x["slots"] < 0)[:, None, None]
        return [_exact_values(t, case["normalize"] and i < 2).masked_fill(dead, 0.0)
                for i, t in enumerate((x["k1"], x["k2"], x["v"]))]
    return _exact_decode(case, seed)
