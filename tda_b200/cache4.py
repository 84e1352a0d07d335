"""The 4-bit paged cache of a serving step: its page plan, writing and reading
it, and attention of one new token a request over it.

    plan = plan_pages(lengths, new_tokens, block_table, free_pages, free_head, page_size, rows)
    cache4_append(cache, k1, k2, v, plan.slots)
    out = cache4_softmax_attention(q1, q2, cache, block_table, plan.lengths, lambda_param)
    out = cache4_threshold_attention(q1, q2, cache, block_table, plan.lengths, beta, lambda_param)

Everything stays on the device and runs on the current stream, nothing is read
back, so a step can be captured in a CUDA graph.  K1, K2 and V are held as
4-bit codes in groups of 32 along the head dimension with a bf16 scale (4.5
bits an element).  There is no CPU fallback, and no gradient: the cache holds
values alone, and a backward through the attention raises.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _lib
from . import ops as _ops
from .sdiff import _CODE, lambda_ref, launch, strides_of, view_of

PAGE_SIZES = (16, 32, 64, 128)


class Cache4:
    """Pages of a differential attention layer's keys and values in 4 bits.

    ``data``: uint8 (num_pages, num_kv_heads, block bytes), zeroed (a slot that
    was never written reads as zeros).  ``normalize_keys``: keys are divided by
    their L2 norm as they are written (the threshold form with normalize)."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda",
                 normalize_keys: bool = False):
        if head_dim not in (64, 128):
            raise ValueError(f"Cache4: head_dim must be 64 or 128, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"Cache4: page_size must be one of {PAGE_SIZES}, got {page_size}")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError("Cache4: num_pages and num_kv_heads must be >= 1")
        if num_pages * page_size >= 1 << 31:
            raise ValueError("Cache4: num_pages * page_size must fit 31 bits")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"Cache4: tda_b200 runs on CUDA tensors only (got device {device}); "
                               "there is no CPU fallback")
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = num_pages, page_size, num_kv_heads, head_dim
        self.normalize_keys = bool(normalize_keys)
        block = _lib.load().tda_cache4_block_bytes(page_size, head_dim)
        self.data = torch.zeros((num_pages, num_kv_heads, block), dtype=torch.uint8, device=device)
        self.device = self.data.device


class PagePlan(NamedTuple):
    """One step's plan, all int32 on the device: per packed row its slot,
    position and request (-1 past the last token; slot -1 too where no page was
    left), prefix sums of the new tokens, tokens held afterwards, the free
    list's new head and the number of tokens that found no page or no row."""
    slots: torch.Tensor
    positions: torch.Tensor
    requests: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    free_head: torch.Tensor
    dropped: torch.Tensor


def _ints(what, name, t, shape, device):
    if type(t) is torch.Tensor and t.dtype is torch.int32 and t.device == device and (shape is None or t.shape == shape):
        return
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} must be an int32 tensor")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} must be on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: {name} must have shape {shape}, got {tuple(t.shape)}")


def _cuda(what, t):
    if type(t) is torch.Tensor and t.is_cuda:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: expected torch.Tensor inputs")
    if not t.is_cuda:
        raise RuntimeError(f"{what}: tda_b200 runs on CUDA tensors only (got device {t.device}); "
                           "there is no CPU fallback")


def _table(what, block_table, requests, device):
    _ints(what, "block_table", block_table, None, device)
    if block_table.dim() != 2 or block_table.shape[0] != requests or block_table.shape[1] < 1:
        raise ValueError(f"{what}: block_table must have shape ({requests}, width >= 1), got {tuple(block_table.shape)}")
    if block_table.stride(1) != 1 or (block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError(f"{what}: block_table rows must be contiguous and apart")
    return block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]


def plan_pages(lengths, new_tokens, block_table, free_pages, free_head, page_size: int, rows: int) -> PagePlan:
    """Pages, slots and positions of one step, built on the device in one launch.

    Request r holds ``lengths[r]`` tokens in the first ceil(lengths / page_size)
    entries of its ``block_table`` row and gets ``new_tokens[r]`` more.  Fresh
    pages are taken from ``free_pages[free_head:]`` in request order and written
    into ``block_table`` in place; the new head is returned, not written back.
    ``rows``: rows of the packed batch of new tokens (its capacity); tokens past
    them take no page, are not in ``lengths`` and count as ``dropped``."""
    what = "plan_pages"
    _cuda(what, lengths)
    dev = lengths.device
    if lengths.dim() != 1 or lengths.shape[0] < 1:
        raise ValueError(f"{what}: lengths must be a vector of at least one request, got {tuple(lengths.shape)}")
    B = lengths.shape[0]
    _ints(what, "lengths", lengths, (B,), dev)
    _ints(what, "new_tokens", new_tokens, (B,), dev)
    _ints(what, "free_head", free_head, (1,), dev)
    _ints(what, "free_pages", free_pages, None, dev)
    if free_pages.dim() != 1:
        raise ValueError(f"{what}: free_pages must be a vector")
    stride = _table(what, block_table, B, dev)
    if page_size < 1:
        raise ValueError(f"{what}: page_size must be >= 1, got {page_size}")
    if rows < 0:
        raise ValueError(f"{what}: rows must be >= 0, got {rows}")
    if not (lengths.is_contiguous() and new_tokens.is_contiguous() and free_pages.is_contiguous()):
        lengths, new_tokens, free_pages = lengths.contiguous(), new_tokens.contiguous(), free_pages.contiguous()
    # one allocation: its parts are views
    buf = torch.empty(3 * rows + 2 * B + 3, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    launch(_lib.load().tda_plan_pages, dev, lengths.data_ptr(), new_tokens.data_ptr(), B, block_table.data_ptr(),
           stride, block_table.shape[1], free_pages.data_ptr(), free_pages.shape[0], free_head.data_ptr(), page_size,
           rows, at, at + 4 * rows, at + 8 * rows, at + 12 * rows, at + 4 * (3 * rows + B + 1),
           at + 4 * (3 * rows + 2 * B + 1), at + 4 * (3 * rows + 2 * B + 2))
    return PagePlan(*buf.split_with_sizes((rows, rows, rows, B + 1, B, 1, 1)))


def _rows(what, cache, slots):
    _cuda(what, slots)
    _ints(what, "slots", slots, None, cache.device)
    if slots.dim() != 1:
        raise ValueError(f"{what}: slots must be a vector, got {tuple(slots.shape)}")
    return slots.contiguous()


def cache4_append(cache: Cache4, k1, k2, v, slots) -> None:
    """Quantise k1, k2, v (tokens, kv heads, head_dim) into ``slots`` (int32; -1
    rows are skipped; slots of one call are distinct).  bf16, fp16 or fp32."""
    what = "cache4_append"
    slots = _rows(what, cache, slots)
    shape = (slots.shape[0], cache.num_kv_heads, cache.head_dim)
    for t in (k1, k2, v):
        _cuda(what, t)
        if t.shape != shape:
            raise ValueError(f"{what}: k1, k2 and v must have shape {shape}, got {tuple(t.shape)}")
        if t.device != cache.device:
            raise RuntimeError(f"{what}: inputs must be on the cache's device")
        if t.dtype not in _CODE or t.dtype != k1.dtype:
            raise TypeError(f"{what}: k1, k2 and v must share one of bf16, fp16, fp32; got {t.dtype}")
    if slots.shape[0] == 0:
        return
    ts = [view_of(t, t.dtype) for t in (k1, k2, v)]
    launch(_lib.load().tda_cache4_append, cache.device, *[t.data_ptr() for t in ts], _CODE[k1.dtype], strides_of(ts),
           slots.data_ptr(), shape[0], cache.data.data_ptr(), cache.num_pages, cache.num_kv_heads, cache.head_dim,
           cache.page_size, int(cache.normalize_keys))


def cache4_read(cache: Cache4, slots, dtype=torch.bfloat16):
    """(k1, k2, v) that ``slots`` hold, (tokens, kv heads, head_dim) in ``dtype``
    (zeros where the slot is -1): what a chunked prefill attends to."""
    what = "cache4_read"
    slots = _rows(what, cache, slots)
    if dtype not in _CODE:
        raise TypeError(f"{what}: dtype must be bf16, fp16 or fp32, got {dtype}")
    shape = (slots.shape[0], cache.num_kv_heads, cache.head_dim)
    out = torch.empty((3, *shape), dtype=dtype, device=cache.device).unbind(0)
    if slots.shape[0] == 0:
        return out
    launch(_lib.load().tda_cache4_read, cache.device, cache.data.data_ptr(), cache.num_pages, cache.num_kv_heads,
           cache.head_dim, cache.page_size, slots.data_ptr(), shape[0], *[t.data_ptr() for t in out], _CODE[dtype])
    return out


@functools.lru_cache(maxsize=256)
def _workspace_size(*sizes) -> int:
    return _lib.load().tda_cache4_workspace_size(*sizes)


class _NoBackward(torch.autograd.Function):
    """``out`` as a result of inputs that want a gradient: asking for it raises
    where an output without a graph would leave it out in silence."""

    @staticmethod
    def forward(ctx, what, out, *inputs):
        ctx.what = what
        return out.detach()

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError(f"{ctx.what} has no backward: it serves from a 4-bit cache (train with "
                           "differential_softmax_attention or differential_threshold_rela_triton)")


def _attend(what, kind, q1, q2, cache, block_table, lengths, lambda_param, scale, beta, relu_power):
    for t in (q1, q2):
        _cuda(what, t)
    if q1.dim() != 3 or q1.shape != q2.shape or q1.shape[2] != cache.head_dim:
        raise ValueError(f"{what}: q1 and q2 must both have shape (batch, heads, {cache.head_dim}), got "
                         f"{tuple(q1.shape)} and {tuple(q2.shape)}")
    B, H, D = q1.shape
    if H == 0 or H % cache.num_kv_heads != 0:
        raise ValueError(f"{what}: the cache's kv heads ({cache.num_kv_heads}) must divide the query heads ({H})")
    if q1.dtype != q2.dtype or q1.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: queries must be bf16 or fp16, got {q1.dtype} and {q2.dtype}")
    dev = cache.device
    if q1.device != dev or q2.device != dev:
        raise RuntimeError(f"{what}: queries must be on the cache's device")
    out = torch.empty((B, H, D), dtype=q1.dtype, device=dev)
    if B == 0:
        return out
    _ints(what, "lengths", lengths, (B,), dev)
    stride = _table(what, block_table, B, dev)
    lengths = lengths.contiguous()
    ts = [view_of(q1, q1.dtype), view_of(q2, q2.dtype)]
    lp, lc, lsb, lsh, lv, keep = lambda_ref(lambda_param, B, H, dev, what)
    width = block_table.shape[1]
    ws_n = _workspace_size(kind, B, H, cache.num_kv_heads, D, cache.page_size, width)
    ws = torch.empty(ws_n, dtype=torch.uint8, device=dev) if ws_n else None
    launch(_lib.load().tda_cache4_attention, dev, kind, ts[0].data_ptr(), ts[1].data_ptr(), _CODE[q1.dtype],
           strides_of(ts), out.data_ptr(), B, H, cache.num_kv_heads, D, cache.data.data_ptr(), cache.num_pages,
           cache.page_size, block_table.data_ptr(), stride, width, lengths.data_ptr(), lp, lc, lsb, lsh, lv, scale,
           beta, relu_power, int(cache.normalize_keys), None if ws is None else ws.data_ptr(), ws_n,
           _ops._status_word(dev).data_ptr())
    if torch.is_grad_enabled() and (q1.requires_grad or q2.requires_grad or
                                    isinstance(lambda_param, torch.Tensor) and lambda_param.requires_grad):
        return _NoBackward.apply(what, out, q1, q2, lambda_param)
    return out


def cache4_softmax_attention(q1, q2, cache: Cache4, block_table, lengths, lambda_param, scale=None):
    """One new token a request: (softmax(scale q1 K1^T) - lambda softmax(scale
    q2 K2^T)) V over the request's ``lengths`` cached tokens, the new one among
    them.  q1, q2: (batch, heads, head_dim) bf16 / fp16; lambda as in
    ``differential_softmax_attention``; a request of length 0 gives zeros.  Not
    differentiable: a backward through it raises."""
    sc = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    if cache.normalize_keys:
        raise ValueError("cache4_softmax_attention: the cache holds normalized keys (made for the threshold form)")
    return _attend("cache4_softmax_attention", _lib.TDA_MAP_SOFTMAX, q1, q2, cache, block_table, lengths, lambda_param,
                   sc, 0.0, 2.0)


def cache4_threshold_attention(q1, q2, cache: Cache4, block_table, lengths, beta, lambda_param, relu_power=2.0):
    """One new token a request in the threshold form: row lengths - 1 of
    ``differential_threshold_rela_triton`` over the cached tokens, (P1 -
    clamp(lambda, 0, 1) P2) V with P = ReLU(q K^T - tau)^p and tau = beta
    sqrt(2 log(lengths) / head_dim); q is L2-normalized when the cache
    normalizes its keys.  ``beta`` and ``relu_power`` are floats (or one-element
    tensors, read on the host).  Not differentiable: a backward through it
    raises."""
    b = float(beta.item()) if isinstance(beta, torch.Tensor) else float(beta)
    p = float(relu_power.item()) if isinstance(relu_power, torch.Tensor) else float(relu_power)
    return _attend("cache4_threshold_attention", _lib.TDA_MAP_THRESHOLD, q1, q2, cache, block_table, lengths,
                   lambda_param, 1.0, b, p)
