"""Softmax differential attention on the tda_b200 C ABI.

``differential_softmax_attention(q1, q2, k1, k2, v, lambda_param, scale=None,
causal=True, key_lengths=None)``:

    out = (softmax(scale q1 k1^T) - lambda softmax(scale q2 k2^T)) v

the form that threshold differential attention replaces, with its gradients
(q1, q2, k1, k2, v and lambda).  q1, q2: (B, H, Sq, D); k1, k2, v: (B, Hkv, Sk,
D), Hkv dividing H (query head h reads kv head h // (H / Hkv); gradients of
shared heads are summed).  Row i sees key j when j < key_lengths[b] and, when
causal, j <= i + Sk - Sq; a row that sees no key gives zeros.  lambda is used
as it is (no clamp): a float, or a tensor that broadcasts over (batch, head).

bf16 and fp16 with head_dim 64 / 128 run on the tcgen05 tensor cores; fp32 and
other head dims (powers of two in [16, 256]) run in fp32 on the CUDA cores;
other float types are widened to fp32.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from . import ops as _ops

_CODE = {torch.float32: _lib.TDA_F32, torch.bfloat16: _lib.TDA_BF16, torch.float16: _lib.TDA_F16}


# Small calls are bound by the host: a stream object costs 2 us to make, its handle alone 0.1.
_raw_stream = torch._C._cuda_getCurrentRawStream
_dispatch_modes = torch._C._len_torch_dispatch_stack


def launch(entry, device: torch.device, *args) -> None:
    """Calls a C entry point on ``device``'s current stream (appended to
    ``args``), making the device current where it is not, and raises on an
    error code."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc)
    if _ops._SYNC_CHECK:
        _ops.check_status(device)


def lambda_ref(lam, B: int, H: int, device: torch.device, what: str):
    """(pointer, dtype code, batch stride, head stride, value, keep-alive) of a
    lambda: a float or one-element CPU tensor is read on the host, a tensor that
    broadcasts over (batch, head) stays on the device in its own type."""
    if not isinstance(lam, torch.Tensor):
        return None, 0, 0, 0, float(lam), None
    if lam.is_cuda and lam.dtype in _CODE and lam.device == device:  # the usual forms, without views
        shape = lam.shape
        if lam.numel() == 1 and len(shape) <= 4:
            return lam.data_ptr(), _CODE[lam.dtype], 0, 0, 0.0, lam
        if len(shape) == 4 and shape[0] == 1 and shape[1] == H and shape[2] == 1 and shape[3] == 1:
            return lam.data_ptr(), _CODE[lam.dtype], 0, lam.stride(1), 0.0, lam
    if not lam.dtype.is_floating_point:
        raise TypeError(f"{what}: lambda must be floating point, got {lam.dtype}")
    if not lam.is_cuda and lam.numel() == 1:
        return None, 0, 0, 0, float(lam.item()), None
    l4 = lam.detach()
    if lam.dim() > 4:
        raise ValueError(f"{what}: lambda may have at most 4 dimensions, got {lam.dim()}")
    l4 = l4[(None,) * (4 - lam.dim())]
    if l4.shape[2] != 1 or l4.shape[3] != 1 or l4.shape[0] not in (1, B) or l4.shape[1] not in (1, H):
        raise ValueError(f"{what}: lambda must broadcast over (batch, head) alone, i.e. to ({B}, {H}, 1, 1); "
                         f"got {tuple(lam.shape)}")
    if l4.device != device:
        l4 = l4.to(device)
    if l4.dtype not in _CODE:
        l4 = l4.float()
    return (l4.data_ptr(), _CODE[l4.dtype], l4.stride(0) if l4.shape[0] != 1 else 0,
            l4.stride(1) if l4.shape[1] != 1 else 0, 0.0, l4)


def _check(q1, q2, k1, k2, v, key_lengths, what="differential_softmax_attention"):
    ts = (q1, q2, k1, k2, v)
    if not all(isinstance(t, torch.Tensor) for t in ts):
        raise TypeError(f"{what}: expected torch.Tensor inputs")
    if q1.dim() != 4 or k1.dim() != 4:
        raise ValueError(f"{what}: expected (batch, heads, seq_len, head_dim) tensors, got {tuple(q1.shape)} and "
                         f"{tuple(k1.shape)}")
    if q1.shape != q2.shape:
        raise ValueError(f"{what}: q1 and q2 must have one shape, got {tuple(q1.shape)} and {tuple(q2.shape)}")
    if not (k1.shape == k2.shape == v.shape):
        raise ValueError(f"{what}: k1, k2 and v must have one shape")
    if q1.shape[0] != k1.shape[0] or q1.shape[3] != k1.shape[3]:
        raise ValueError(f"{what}: batch and head_dim of queries {tuple(q1.shape)} and keys {tuple(k1.shape)} differ")
    if k1.shape[1] == 0 or q1.shape[1] % k1.shape[1] != 0:
        raise ValueError(f"{what}: the kv heads ({k1.shape[1]}) must divide the query heads ({q1.shape[1]})")
    D = q1.shape[3]
    if D < 16 or D > 256 or (D & (D - 1)) != 0:
        raise ValueError(f"{what}: head_dim must be a power of two in [16, 256], got {D}")
    if not q1.is_cuda:
        raise RuntimeError(f"{what}: tda_b200 runs on CUDA tensors only (got device {q1.device}); "
                           "there is no CPU fallback")
    dev, dt = q1.device, q1.dtype
    for t in ts:
        if t.device != dev:
            raise RuntimeError(f"{what}: all inputs must be on one device")
        if not (t.dtype is dt and dt in _CODE) and not t.dtype.is_floating_point:
            raise TypeError(f"{what}: floating point inputs required, got {t.dtype}")
    if key_lengths is not None:
        if not isinstance(key_lengths, torch.Tensor) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what}: key_lengths must be an int32 or int64 tensor")
        if key_lengths.shape != (q1.shape[0],):
            raise ValueError(f"{what}: key_lengths must have shape ({q1.shape[0]},), got {tuple(key_lengths.shape)}")
        if key_lengths.device != q1.device:
            raise RuntimeError(f"{what}: key_lengths must be on the inputs' device")


def _check_saved(q1, dout, o12, lse, what="differential_softmax_attention backward"):
    """What the backward kernels read besides the inputs: by pointer, so a wrong
    shape, type or device would be read out of bounds."""
    B, H, Sq, D = q1.shape
    for name, t, shape in (("dout", dout, (B, H, Sq, D)), ("o12", o12, (2, B, H, Sq, D)), ("lse", lse, (2, B, H, Sq))):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a tensor, got {type(t).__name__}")
        if t.shape != shape:
            raise ValueError(f"{what}: {name} must have shape {shape}, got {tuple(t.shape)}")
        if t.device != q1.device:
            raise RuntimeError(f"{what}: {name} must be on the inputs' device, got {t.device}")
        if not (t.dtype.is_floating_point if t is dout else t.dtype == torch.float32 and t.is_contiguous()):
            raise TypeError(f"{what}: {name} must be {'floating point' if t is dout else 'contiguous fp32'}, got {t.dtype}")


def _compute_dtype(ts) -> torch.dtype:
    common = ts[0].dtype
    for t in ts[1:]:
        if t.dtype is not common:
            common = torch.promote_types(common, t.dtype)
    return common if common in _CODE else torch.float32


def view_of(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``t`` in ``dtype`` as the kernels read it in place: contiguous last
    dimension, other strides positive multiples of 8 elements (any stride of a
    dimension of size 1 counts as fitting), 16-byte aligned; else a copy."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    if ok:
        for n, s in zip(t.shape[:-1], t.stride()[:-1]):
            if n != 1 and (s <= 0 or s % 8):
                ok = False
                break
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def strides_of(ts):
    """Element strides of all but the last dimension, a stride that is never
    used (size 1) given as the row's length; None when all are contiguous."""
    if all(t.is_contiguous() for t in ts):
        return None
    out = []
    for t in ts:
        d = t.shape[-1]
        out += [s if n != 1 else d for n, s in zip(t.shape[:-1], t.stride()[:-1])]
    return (ctypes.c_int64 * len(out))(*out)


def _lengths32(key_lengths):
    if key_lengths is None or (key_lengths.dtype == torch.int32 and key_lengths.is_contiguous()):
        return key_lengths
    return key_lengths.to(torch.int32).contiguous()


def sdiff_forward(q1, q2, k1, k2, v, lambda_param, scale=None, causal=True, key_lengths=None, save=True):
    """(out, o12, lse): the attention and, where ``save``, what its backward
    needs: each map's product with v (fp32 (2, B, H, Sq, D)) and the row sums
    (fp32 (2, B, H, Sq), log2; +inf where a row sees no key); None otherwise.
    No autograd."""
    _check(q1, q2, k1, k2, v, key_lengths)
    B, H, Sq, D = q1.shape
    Hkv, Sk = k1.shape[1], k1.shape[2]
    dt = _compute_dtype((q1, q2, k1, k2, v))
    out = torch.empty((B, H, Sq, D), dtype=dt, device=q1.device)
    o12 = torch.empty((2, B, H, Sq, D), dtype=torch.float32, device=q1.device) if save else None
    lse = torch.empty((2, B, H, Sq), dtype=torch.float32, device=q1.device) if save else None
    if out.numel() == 0 or Sk == 0:
        return out.zero_(), o12.zero_() if save else None, lse.fill_(math.inf) if save else None
    ts = [view_of(t, dt) for t in (q1, q2, k1, k2, v)]
    kl = _lengths32(key_lengths)
    lp, lc, lsb, lsh, lv, keep = lambda_ref(lambda_param, B, H, q1.device, "differential_softmax_attention")
    launch(_lib.load().tda_sdiff_fwd, q1.device, *[t.data_ptr() for t in ts], strides_of(ts), out.data_ptr(),
           o12.data_ptr() if save else None, lse.data_ptr() if save else None, _CODE[dt], B, H, Hkv, Sq, Sk, D,
           1.0 / math.sqrt(D) if scale is None else float(scale), int(causal), None if kl is None else kl.data_ptr(),
           lp, lc, lsb, lsh, lv, _ops._status_word(q1.device).data_ptr())
    return out, o12, lse


def sdiff_backward(q1, q2, k1, k2, v, dout, o12, lse, lambda_param, scale=None, causal=True, key_lengths=None,
                   need_dlam=True):
    """(dq1, dq2, dk1, dk2, dv, dlam) for the upstream gradient ``dout`` from
    the forward's (o12, lse); gradients in the compute type, ``dlam`` fp32 (B,
    H), None when not asked for."""
    _check(q1, q2, k1, k2, v, key_lengths)
    _check_saved(q1, dout, o12, lse)
    B, H, Sq, D = q1.shape
    Hkv, Sk = k1.shape[1], k1.shape[2]
    dt = _compute_dtype((q1, q2, k1, k2, v))
    dev = q1.device
    dq = [torch.empty((B, H, Sq, D), dtype=dt, device=dev) for _ in range(2)]
    dkv = [torch.empty((B, Hkv, Sk, D), dtype=dt, device=dev) for _ in range(3)]
    dlam = torch.empty((B, H), dtype=torch.float32, device=dev) if need_dlam else None
    if q1.numel() == 0 or Sk == 0:
        return (*[t.zero_() for t in dq + dkv], dlam.zero_() if need_dlam else None)
    ts = [view_of(t, dt) for t in (q1, q2, k1, k2, v)]
    g = view_of(dout, dt)
    kl = _lengths32(key_lengths)
    lp, lc, lsb, lsh, lv, keep = lambda_ref(lambda_param, B, H, dev, "differential_softmax_attention")
    lib = _lib.load()
    ws_n = lib.tda_sdiff_bwd_workspace_size(B, H, Sq)
    ws = torch.empty(ws_n, dtype=torch.uint8, device=dev)
    launch(lib.tda_sdiff_bwd, dev, *[t.data_ptr() for t in ts], strides_of(ts), g.data_ptr(), strides_of([g]),
           o12.data_ptr(), lse.data_ptr(), *[t.data_ptr() for t in dq + dkv], dlam.data_ptr() if need_dlam else None,
           _CODE[dt], B, H, Hkv, Sq, Sk, D, 1.0 / math.sqrt(D) if scale is None else float(scale), int(causal),
           None if kl is None else kl.data_ptr(), lp, lc, lsb, lsh, lv, ws.data_ptr(), ws_n,
           _ops._status_word(dev).data_ptr())
    return (*dq, *dkv, dlam)


def dlam_like(dlam: torch.Tensor, lam: torch.Tensor) -> torch.Tensor:
    """(B, H) gradients summed to lambda's shape, in its type and on its device."""
    g = dlam[:, :, None, None]
    if lam.numel() == 1:
        g = g.sum()
    else:
        g = g.sum_to_size((1,) * (4 - lam.dim()) + tuple(lam.shape))
    return g.reshape(lam.shape).to(device=lam.device, dtype=lam.dtype)


class DifferentialSoftmaxFunction(torch.autograd.Function):
    """forward(q1, q2, k1, k2, v, lambda_param, scale, causal, key_lengths)."""

    @staticmethod
    def forward(ctx, q1, q2, k1, k2, v, lambda_param, scale, causal, key_lengths):
        out, o12, lse = sdiff_forward(q1, q2, k1, k2, v, lambda_param, scale, causal, key_lengths)
        lam_t = lambda_param if isinstance(lambda_param, torch.Tensor) else None
        ctx.save_for_backward(q1, q2, k1, k2, v, lam_t, key_lengths, o12, lse)
        ctx.lam = None if lam_t is not None else float(lambda_param)
        ctx.scale, ctx.causal = scale, causal
        return out if out.dtype == q1.dtype else out.to(q1.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q1, q2, k1, k2, v, lam_t, kl, o12, lse = ctx.saved_tensors
        lam = ctx.lam if lam_t is None else lam_t
        need = lam_t is not None and ctx.needs_input_grad[5]
        g = sdiff_backward(q1, q2, k1, k2, v, dout, o12, lse, lam, ctx.scale, ctx.causal, kl, need)
        cast = [x if x.dtype == t.dtype else x.to(t.dtype) for x, t in zip(g[:5], (q1, q2, k1, k2, v))]
        return (*cast, dlam_like(g[5], lam_t) if need else None, None, None, None)


def _wants_grad(*ts) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    return False


def _traced(q1) -> bool:
    """Whether the call is recorded or run without data (torch.compile, make_fx,
    fake and meta tensors, dispatch modes): then it is the registered operator.
    A plain call goes past it: small calls are bound by the host."""
    if torch.compiler.is_compiling() or _dispatch_modes():
        return True
    kind = type(q1)
    return q1.is_meta if kind is torch.Tensor or kind is torch.nn.Parameter else isinstance(q1, torch.Tensor)


def differential_softmax_attention(q1, q2, k1, k2, v, lambda_param, scale=None, causal=True, key_lengths=None):
    """out = (softmax(scale q1 k1^T) - lambda softmax(scale q2 k2^T)) v, q1's
    shape and dtype; differentiable in q1, q2, k1, k2, v and lambda.  ``scale``
    defaults to head_dim ** -0.5.  See the module's docstring.  Where it is
    traced (torch.compile, make_fx, fake tensors) it is the operator
    ``tda::sdiff_fwd``."""
    if _traced(q1):
        lam = lambda_param if isinstance(lambda_param, torch.Tensor) else torch.tensor(float(lambda_param))
        sc = 1.0 / math.sqrt(q1.shape[-1]) if scale is None else float(scale)
        return torch.ops.tda.sdiff_fwd(q1, q2, k1, k2, v, lam, sc, bool(causal), key_lengths,
                                       _wants_grad(q1, q2, k1, k2, v, lambda_param))[0]
    if not _wants_grad(q1, q2, k1, k2, v, lambda_param):
        out = sdiff_forward(q1, q2, k1, k2, v, lambda_param, scale, causal, key_lengths, save=False)[0]
        return out if out.dtype == q1.dtype else out.to(q1.dtype)
    return DifferentialSoftmaxFunction.apply(q1, q2, k1, k2, v, lambda_param, scale, causal, key_lengths)
