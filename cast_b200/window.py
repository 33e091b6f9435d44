"""Sliding-window attention with visible first tokens (sinks).

Beside the block-sparse attention of :mod:`cast_b200.rcsa`, which attends to
chosen key blocks, these attend to the newest keys of a session and its first
ones -- what a streaming rollout keeps -- densely:

* :func:`window_attention` -- a chunk of queries (or one) over dense keys;
* :func:`paged_window_attention` -- a few new tokens of many sessions over a
  paged cache (:func:`cast_b200.rotary.qk_norm_rope` writes it).

Query i of Lq is at position ``p = kv_len - Lq + i`` of its session and sees
key ``j < kv_len`` where ``f(j) <= f(p)`` and (``f(j) > f(p) - window`` or
``f(j) < sinks``), ``f(x) = x // frame_tokens``: with ``frame_tokens=1``
causal over the last ``window`` tokens, its own among them, and the first
``sinks``; with the tokens of a latent frame, block-causal over frames.

Every function runs CUDA kernels of ``libcast_b200.so`` on the current stream
of the tensors' device.  They have no gradient: inputs that need one are
refused.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .rotary import DTYPES, _check, _check_out, _keep, _launch, _refuse_gradients, _sig, _strides

_TYPES = (torch.bfloat16, torch.float16)
_Twelve = ctypes.c_longlong * 12
_FOREVER = 1 << 40
_plans: dict = {}
_paged_plans: dict = {}


def _options(window, sinks, frame_tokens):
    """The options as the numbers they are now (they may be given as tensors)."""
    return None if window is None else int(window), int(sinks), int(frame_tokens)


def _rule(window, sinks, frame_tokens):
    window = _FOREVER if window is None else window
    if window < 1 or sinks < 0 or frame_tokens < 1:
        raise ValueError("window must be at least 1 (or None), sinks at least 0, frame_tokens at least 1")
    # (no session has 2^30 keys: a longer frame is one that holds them all)
    return min(window, _FOREVER), min(sinks, _FOREVER), min(frame_tokens, 1 << 30)


def _workspace_bytes(name: str, device: torch.device, *shape) -> int:
    """Bytes of scratch memory of one call.  Each call takes a buffer of its
    own (stream-ordered: the allocator hands it on when the call's work is
    done), so calls on several streams and captured graphs never share one."""
    with torch.cuda.device(device):
        return int(getattr(_lib.load(), name)(*shape))


def _lens(kv_lens, b, device):
    _check("kv_lens", kv_lens, 1, (torch.int32,), device)
    if kv_lens.numel() != b or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be a contiguous int32 [{b}]")


def _heads(q, k, hk):
    if q.shape[1] % max(hk, 1) or hk == 0:
        raise ValueError(f"{q.shape[1]} query heads do not share {hk} key heads evenly")
    if q.shape[3] not in (64, 128) or k.shape[3] != q.shape[3]:
        raise ValueError(f"head vectors of 64 or 128 values, the same for all; got {q.shape[3]} and {k.shape[3]}")


def _window_plan(q, k, v, window, sinks, frame_tokens, kv_lens, out):
    _check("q", q, 4, _TYPES)
    dev = q.device
    _check("k", k, 4, (q.dtype,), dev)
    _check("v", v, 4, (q.dtype,), dev)
    b, hq, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    _heads(q, k, hk)
    if k.shape[0] != b or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if kv_lens is not None:
        _lens(kv_lens, b, dev)
    rule = _rule(window, sinks, frame_tokens)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_out("out", out, q.shape, q.dtype, dev)
    if q.numel() == 0 or lk == 0:
        return q.numel() == 0, lk == 0, dev.index, 0, 0.0, (), ()
    shape = (b, hq, hk, lq, lk, d)
    n = _workspace_bytes("cast_window_attention_workspace_bytes", dev, *shape, *rule)
    order = (0, 1, 2)
    strides = _Twelve(*_strides(q, order), *_strides(k, order), *_strides(v, order), *_strides(out, order))
    return False, False, dev.index, n, 1.0 / math.sqrt(d), DTYPES[q.dtype], (*shape, strides, *rule)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None, sinks: int = 0,
                     frame_tokens: int = 1, kv_lens: torch.Tensor | None = None, sm_scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``q`` ``[B,Hq,Lq,D]`` over ``k``, ``v`` ``[B,Hk,Lk,D]``
    (bf16 or fp16, D 64 or 128, Hq a multiple of Hk, any strides on 16-byte
    boundaries with dense head vectors) by the rule of the module's text.

    ``window=None``: every earlier key.  ``kv_lens``: int32 ``[B]``, the keys
    of each session (default Lk; the queries are its last Lq positions, and
    rows of k and v behind them are never used, whatever they hold).
    ``sm_scale`` defaults to ``1/sqrt(D)``.  Returns ``[B,Hq,Lq,D]`` (``out``
    may be ``q``; it must not overlap k or v); a query that sees nothing gives
    zeros, one that sees a NaN score NaN.  A length outside ``[0, Lk]`` is clipped
    and sets the device error word.
    """
    window, sinks, frame_tokens = _options(window, sinks, frame_tokens)
    try:
        key = (q.dtype, q.shape, q.stride(), q.device, k.dtype, k.shape, k.stride(), k.device, v.dtype, v.shape,
               v.stride(), v.device,
               None if kv_lens is None else (kv_lens.dtype, kv_lens.shape, kv_lens.stride(), kv_lens.device),
               None if out is None else _sig(out),
               window, sinks, frame_tokens)
        plan = _plans.get(key)
    except AttributeError:
        key = plan = None  # (not a tensor: the checks say so)
    if plan is None:
        plan = _keep(_plans, key, _window_plan(q, k, v, window, sinks, frame_tokens, kv_lens, out))
    empty, blind, index, nbytes, scale, dtype, rest = plan
    _refuse_gradients(q, k, v, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if empty:
        return out
    if blind:
        return out.zero_()
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(index, "cast_window_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype,
            None if kv_lens is None else kv_lens.data_ptr(), *rest, scale if sm_scale is None else sm_scale,
            out.data_ptr(), _lib.ptr(ws), nbytes)
    return out


def _paged_plan(q, k_pages, v_pages, block_table, kv_lens, window, sinks, frame_tokens, out):
    _check("q", q, 4, _TYPES)
    dev = q.device
    _check("k_pages", k_pages, 4, (q.dtype,), dev)
    _check("v_pages", v_pages, 4, (q.dtype,), dev)
    b, hq, lq, d = q.shape
    pages, hk, page, _ = k_pages.shape
    _heads(q, k_pages, hk)
    if v_pages.shape != k_pages.shape:
        raise ValueError(f"v_pages {tuple(v_pages.shape)} differs from k_pages {tuple(k_pages.shape)}")
    _check("block_table", block_table, 2, (torch.int32,), dev)
    if block_table.shape[0] != b or not block_table.is_contiguous():
        raise ValueError(f"block_table must be a contiguous int32 [{b}, max_pages], got {tuple(block_table.shape)}")
    _lens(kv_lens, b, dev)
    rule = _rule(window, sinks, frame_tokens)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_out("out", out, q.shape, q.dtype, dev)
    max_pages = block_table.shape[1]
    if q.numel() == 0 or max_pages * pages * page == 0:
        return q.numel() == 0, max_pages * pages * page == 0, dev.index, 0, 0.0, (), (), ()
    n = _workspace_bytes("cast_paged_window_attention_workspace_bytes", dev, b, hq, hk, lq, d, page, max_pages, *rule)
    order = (0, 1, 2)
    strides = _Twelve(*_strides(q, order), *_strides(k_pages, order), *_strides(v_pages, order), *_strides(out, order))
    return (False, False, dev.index, n, 1.0 / math.sqrt(d), DTYPES[q.dtype], (max_pages, pages, page),
            (b, hq, hk, lq, d, strides, *rule))


def paged_window_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                           kv_lens: torch.Tensor, *, window: int | None, sinks: int = 0, frame_tokens: int = 1,
                           sm_scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`window_attention` of a few new tokens over a paged cache.

    Key j of session b is row ``j % page`` of page ``block_table[b, j //
    page]`` (int32 ``[B, max_pages]``) of ``k_pages``, ``v_pages``
    ``[n_pages,Hk,page,D]``; ``kv_lens`` int32 ``[B]`` counts the new tokens,
    whose keys and values are in the cache already.  Entries of pages that no
    query sees are not read, so pages that left the window may be given away.
    An entry outside ``[0, n_pages)`` that is seen hides its keys and sets the
    device error word, as a length outside ``[0, max_pages * page]`` does.
    Sessions may share pages (a common prefix).
    """
    window, sinks, frame_tokens = _options(window, sinks, frame_tokens)
    try:
        key = (q.dtype, q.shape, q.stride(), q.device, k_pages.dtype, k_pages.shape, k_pages.stride(), k_pages.device,
               v_pages.dtype, v_pages.shape, v_pages.stride(), v_pages.device, block_table.dtype, block_table.shape,
               block_table.stride(), block_table.device, kv_lens.dtype, kv_lens.shape, kv_lens.stride(),
               kv_lens.device,
               None if out is None else _sig(out), window, sinks, frame_tokens)
        plan = _paged_plans.get(key)
    except AttributeError:
        key = plan = None  # (not a tensor: the checks say so)
    if plan is None:
        plan = _keep(_paged_plans, key, _paged_plan(q, k_pages, v_pages, block_table, kv_lens, window, sinks,
                                                    frame_tokens, out))
    empty, blind, index, nbytes, scale, dtype, pages, rest = plan
    _refuse_gradients(q, k_pages, v_pages, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if empty:
        return out
    if blind:
        return out.zero_()
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch(index, "cast_paged_window_attention", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), dtype,
            block_table.data_ptr(), *pages, kv_lens.data_ptr(), *rest, scale if sm_scale is None else sm_scale,
            out.data_ptr(), _lib.ptr(ws), nbytes)
    return out
