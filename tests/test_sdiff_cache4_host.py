"""Refusals of the softmax differential and 4-bit cache entry points, on the CPU."""
import pytest
import torch

import tda_b200
from tda_b200 import _lib


def _fwd(lib, **kw):
    a = dict(q=16, strides=None, out=16, o12=16, lse=16, dtype=_lib.TDA_BF16, B=1, H=2, Hkv=1, Sq=8, Sk=8, D=64, scale=0.1,
             lam=None, lc=0, lsb=0, status=16)
    a.update(kw)
    return lib.tda_sdiff_fwd(a["q"], 16, 16, 16, 16, a["strides"], a["out"], a["o12"], a["lse"], a["dtype"], a["B"], a["H"],
                             a["Hkv"], a["Sq"], a["Sk"], a["D"], a["scale"], 1, None, a["lam"], a["lc"], a["lsb"], 0, 0.5,
                             a["status"], None)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q=8), dict(out=None), dict(lse=None), dict(o12=None), dict(o12=8), dict(status=None), dict(dtype=9), dict(B=0), dict(Sq=0),
    dict(Sk=0), dict(H=3, Hkv=2), dict(Hkv=0), dict(D=48), dict(D=512), dict(D=8), dict(scale=0.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(lam=16, lc=7), dict(lam=16, lc=0, lsb=-1),
    dict(B=1 << 30, H=1 << 10), dict(Sq=1 << 31),
])
def test_forward_refuses(kw):
    lib = _lib.load()
    assert _fwd(lib, **kw) == _lib.TDA_ERR_INVALID
    assert lib.tda_last_error()


def test_forward_refuses_strides():
    import ctypes
    lib = _lib.load()
    good = [512, 64 * 8, 64] * 5
    for at, bad in ((0, 0), (4, -8), (8, 4), (14, 63)):
        s = list(good)
        s[at] = bad
        assert _fwd(lib, strides=(ctypes.c_int64 * 15)(*s)) == _lib.TDA_ERR_INVALID


def test_backward_refuses():
    lib = _lib.load()
    ws = lib.tda_sdiff_bwd_workspace_size(2, 3, 100)
    assert ws == 2 * 2 * 3 * 128 * 72 and lib.tda_sdiff_bwd_workspace_size(0, 3, 100) == 0

    def call(dout=16, ds=None, dq=16, lse=16, w=16, n=2 * 2 * 128 * 72):
        return lib.tda_sdiff_bwd(16, 16, 16, 16, 16, None, dout, ds, 16, lse, dq, 16, 16, 16, 16, None, _lib.TDA_BF16, 1,
                                 2, 1, 8, 8, 64, 0.1, 1, None, None, 0, 0, 0, 0.5, w, n, 16, None)
    assert call(dout=None) == call(dq=8) == call(lse=None) == _lib.TDA_ERR_INVALID
    assert call(w=None) == call(n=10) == call(w=8) == _lib.TDA_ERR_WORKSPACE


def test_cache_entries_refuse():
    lib = _lib.load()
    assert lib.tda_cache4_block_bytes(64, 128) == 3 * 64 * (64 + 8) and lib.tda_cache4_block_bytes(16, 64) == 3 * 16 * 36
    assert lib.tda_cache4_block_bytes(24, 128) == lib.tda_cache4_block_bytes(64, 96) == lib.tda_cache4_block_bytes(8, 64) == 0

    def append(k=16, slots=16, T=4, cache=16, pages=4, H=2, D=64, page=16, dtype=_lib.TDA_BF16):
        return lib.tda_cache4_append(k, 16, 16, dtype, None, slots, T, cache, pages, H, D, page, 0, None)
    assert append(D=96) == _lib.TDA_ERR_UNSUPPORTED
    for kw in (dict(k=None), dict(k=8), dict(slots=None), dict(T=0), dict(cache=None), dict(cache=8), dict(pages=0),
               dict(H=0), dict(page=20), dict(dtype=5), dict(pages=1 << 28)):
        assert append(**kw) == _lib.TDA_ERR_INVALID, kw

    def attend(map=0, q=16, dtype=_lib.TDA_BF16, B=1, H=2, Hkv=1, D=64, table=16, stride=4, width=4, lens=16, scale=0.1,
               power=2.0, out=16, status=16):
        return lib.tda_cache4_attention(map, q, 16, dtype, None, out, B, H, Hkv, D, 16, 4, 16, table, stride, width, lens,
                                        None, 0, 0, 0, 0.5, scale, 1.0, power, 0, None, 0, status, None)
    assert attend(dtype=_lib.TDA_F32) == _lib.TDA_ERR_UNSUPPORTED and attend(D=32) == _lib.TDA_ERR_UNSUPPORTED
    for kw in (dict(map=2), dict(q=None), dict(q=4), dict(out=None), dict(B=0), dict(B=70000), dict(H=3, Hkv=2), dict(table=None),
               dict(stride=2), dict(width=0), dict(lens=None), dict(status=None), dict(scale=-1.0), dict(map=1, power=float("nan")),
               dict(width=1 << 28, stride=1 << 28)):
        assert attend(**kw) == _lib.TDA_ERR_INVALID, kw
    assert attend(width=1 << 12, stride=1 << 12) == _lib.TDA_ERR_WORKSPACE
    assert lib.tda_cache4_workspace_size(0, 1, 2, 1, 64, 16, 1 << 12) > 0

    def plan(lens=16, B=2, width=4, stride=4, page=16, rows=8, slots=16, nfree=4, free=16):
        return lib.tda_plan_pages(lens, 16, B, 16, stride, width, free, nfree, 16, page, rows, slots, 16, 16, 16, 16, 16, 16, None)
    for kw in (dict(lens=None), dict(B=0), dict(width=0), dict(stride=3), dict(page=0), dict(rows=-1), dict(slots=None),
               dict(nfree=-1), dict(free=None), dict(width=1 << 28, stride=1 << 28)):
        assert plan(**kw) == _lib.TDA_ERR_INVALID, kw


def test_python_refusals():
    q = torch.zeros(1, 2, 8, 64)
    k = torch.zeros(1, 1, 8, 64)
    f = tda_b200.differential_softmax_attention
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        f(q, q, k, k, k, 0.5)
    with pytest.raises(ValueError, match="one shape"):
        f(q, q[:, :1], k, k, k, 0.5)
    with pytest.raises(ValueError, match="one shape"):
        f(q, q, k, k, k[:, :, :4], 0.5)
    with pytest.raises(ValueError, match="divide"):
        f(torch.zeros(1, 3, 8, 64), torch.zeros(1, 3, 8, 64), *[torch.zeros(1, 2, 8, 64)] * 3, 0.5)
    with pytest.raises(ValueError, match="head_dim"):
        f(*[torch.zeros(1, 2, 8, 48)] * 5, 0.5)
    with pytest.raises(ValueError, match="seq_len"):
        f(*[torch.zeros(2, 8, 64)] * 5, 0.5)
    with pytest.raises(TypeError):
        f(q, q, k, k, None, 0.5)
    with pytest.raises(ValueError, match="broadcast"):
        tda_b200.sdiff.lambda_ref(torch.zeros(1, 2, 8, 1), 1, 2, torch.device("cpu"), "x")
    with pytest.raises(TypeError):
        tda_b200.sdiff.lambda_ref(torch.zeros(2, dtype=torch.int32), 1, 2, torch.device("cpu"), "x")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tda_b200.Cache4(4, 16, 2, 64, "cpu")
    for bad in (dict(head_dim=96), dict(page_size=24), dict(num_pages=0), dict(num_kv_heads=0)):
        with pytest.raises(ValueError):
            tda_b200.Cache4(**{**dict(num_pages=4, page_size=16, num_kv_heads=2, head_dim=64), **bad})
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        tda_b200.plan_pages(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], 16, 2)


def test_trace_without_a_gpu():
    """The operators' shapes under fake tensors (what torch.compile sees)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = torch.empty(2, 4, 7, 64, dtype=torch.bfloat16), torch.empty(2, 2, 9, 64, dtype=torch.bfloat16)
        lam = torch.empty(1, 4, 1, 1)
        out, o12, lse = torch.ops.tda.sdiff_fwd(q, q, k, k, k, lam, 0.1, True, None)
        assert out.shape == q.shape and o12.shape == (2, 2, 4, 7, 64) and o12.dtype == torch.float32 and lse.shape == (2, 2, 4, 7) and lse.dtype == torch.float32
        g = torch.ops.tda.sdiff_bwd(q, q, k, k, k, q, o12, lse, lam, 0.1, True, None, True)
        assert [x.shape for x in g] == [q.shape, q.shape, k.shape, k.shape, k.shape, lam.shape]
