"""Rotary positions, and the norm of query and key heads with the rotation.

* :func:`rope_frequencies` / :func:`rope_table` -- the angles of one position
  step for each pair (one axis or three, scaled for long contexts), and the
  (cos, sin) table that the kernels read.
* :func:`rope` -- turns the pairs of a tensor's heads by their positions.
* :func:`qk_norm_rope` -- RMS norm of the query and key heads of a projection
  and the rotation, one launch for both; with a paged cache the keys and
  values go straight to their slots
  (:func:`cast_b200.window.paged_window_attention` reads them).

The complex phase of the reference's compact layout (``[L, D/2]``,
``proposed/matrix_curvature_phase_frame_weave.py:5484-5563``) is a table with
one row a token: ``compact.phase_pairs(phase)[:, 0]`` with positions
``0..L-1``.

Every function but the two that make the table runs CUDA kernels of
``libcast_b200.so`` on the current stream of the tensors' device.  They have
no gradient: inputs that need one are refused.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_POSITION_TYPES = (torch.int32, torch.int64)
_Six, _Fifteen, _Three = ctypes.c_longlong * 6, ctypes.c_longlong * 15, ctypes.c_int * 3


def _check(name: str, t, ndim: int, dtypes, device=None) -> None:
    """A CUDA tensor of the given rank and types whose last dimension is dense."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU implementation)")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got shape {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")


def _check_out(name: str, t, shape, dtype, device) -> None:
    _check(name, t, len(shape), (dtype,), device)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    # places of the dimensions, from the densest: none may run into the next
    reach = 0
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            raise ValueError(f"{name}: elements share memory (strides {t.stride()})")
        reach += stride * (n - 1)


def _strides(t: torch.Tensor, order) -> list[int]:
    """Strides of the given dimensions; 0 where a dimension has one element
    (its stride is never used and may be anything)."""
    shape, stride = t.shape, t.stride()
    return [stride[d] if shape[d] > 1 else 0 for d in order]


# Checked calls, by all that their checks look at (types, shapes, strides,
# devices, options; no tensor, address or value): a call like an earlier one
# is launched without checking it again.  Options enter as the numbers they
# are at the call: a tensor would be found again after its value has changed.
_PLANS_KEPT = 4096
_fn: dict[str, object] = {}


def _sig(t):
    return None if t is None else (t.dtype, t.shape, t.stride(), t.device)


def _keep(plans: dict, key, plan):
    if len(plans) >= _PLANS_KEPT:
        plans.clear()
    plans[key] = plan
    return plan


def _refuse_gradients(*tensors) -> None:
    """No input may need a gradient, of reverse or of forward mode (a tangent
    passes ``torch.no_grad``), and none may be asked of an output given."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("an input or out needs a gradient, which this operator has not (use torch.no_grad())")
    if forward_ad._current_level >= 0:  # (tensors have tangents within a dual level alone)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("an input or out has a tangent (forward-mode gradient), which this operator has not")


def _launch(index: int, name: str, *args) -> None:
    """Calls an entry point on the current stream of device ``index``, which
    is made current for the call."""
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(_lib.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream)
    if status:
        _lib.check(status, name)


def rope_frequencies(rotary_dim: int, *, base: float = 10000.0, axes=None, scaling=None) -> torch.Tensor:
    """float64 ``[rotary_dim / 2]``: the angle of one position step of each pair.

    One axis: ``base ** (-2j / rotary_dim)``.  ``axes`` (pairs of each axis,
    their sum ``rotary_dim / 2``): pair i of an axis of n pairs turns by
    ``base ** (-i / n)``.  ``scaling`` stretches the positions the angles were
    learned for:

    * ``("linear", f)``: every step divided by ``f``;
    * ``("ntk", f)``: the base raised by ``f ** (d / (d - 2))``, d twice the
      axis' pairs, so that the slowest pair is stretched ``f`` times and the
      fastest not at all;
    * ``("yarn", f, length)`` or ``("yarn", f, length, fast, slow)``: a pair
      that turns more than ``fast`` (32) times over the ``length`` learned
      positions keeps its step, one that turns less than ``slow`` (1) times is
      divided by ``f``, the pairs between blend linearly in their index (from
      the last whole index that is kept to the first that is divided, which may
      lie past the last pair, at the axis' last value at most).
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if not base > 1.0:
        raise ValueError("base must be above 1")
    parts = [rotary_dim // 2] if axes is None else [int(n) for n in axes]
    if sum(parts) != rotary_dim // 2 or min(parts) < 0:
        raise ValueError(f"axes {axes} must add up to {rotary_dim // 2} pairs")
    kind, factor, rest = (None, 1.0, ()) if scaling is None else (scaling[0], float(scaling[1]), tuple(scaling[2:]))
    if kind not in (None, "linear", "ntk", "yarn") or not factor > 0.0 \
            or (kind == "yarn" and len(rest) in (0, 2)):
        raise ValueError(f"scaling {scaling!r}: ('linear' | 'ntk', factor) or ('yarn', factor, length[, fast, slow])")
    if kind == "yarn":
        length, fast, slow = map(float, (*rest, 32.0, 1.0) if len(rest) == 1 else rest[:3])
        if not (0.0 < length < math.inf and 0.0 < slow <= fast < math.inf):
            raise ValueError(f"scaling {scaling!r}: length and slow must be positive, fast not below slow")
    out = []
    for n in parts:
        i = torch.arange(n, dtype=torch.float64)
        b = base * factor ** (n / (n - 1)) if kind == "ntk" and n > 1 else base
        f = torch.pow(torch.tensor(b, dtype=torch.float64), -i / max(n, 1))
        if kind == "linear":
            f = f / factor
        elif kind == "yarn":
            def pair_of(turns):  # the (fractional) pair that turns so often over the learned length
                return n * math.log(length / (turns * 2 * math.pi)) / math.log(base)

            # (places run to the head's 2 n values, past the last pair: there the ramp of a
            # long learned length ends, and no pair is divided by the whole factor)
            lo = max(math.floor(pair_of(fast)), 0)
            hi = min(math.ceil(pair_of(slow)), max(2 * n - 1, 0))
            blend = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)  # 0: kept, 1: divided
            if pair_of(slow) <= 0:  # a length that no pair turns over so often
                blend = torch.ones_like(i)
            f = f * (1.0 - blend) + f / factor * blend
        out.append(f)
    return torch.cat(out)


def rope_table(frequencies: torch.Tensor, positions: int, *, amplitude: float = 1.0, device=None) -> torch.Tensor:
    """float32 ``[positions, pairs, 2]``: (cos, sin) of every position and pair,
    from angles in 64 bits, times ``amplitude`` (long-context scalings raise
    the logits with it).  Made once and kept, as a weight is."""
    if positions <= 0:
        raise ValueError("positions must be positive")
    dev = torch.device(device if device is not None else "cuda")
    f = frequencies.to(device=dev, dtype=torch.float64)
    angle = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * f
    return (torch.stack([angle.cos(), angle.sin()], -1) * float(amplitude)).float().contiguous()


def _turns(table, positions, axes, b, l, d, interleaved, inverse, start, device):
    """Checked arguments of the rotation: ``(rows, 64 bit, batch stride, first,
    axes), R, flags``."""
    flags = (1 if interleaved else 0) | (2 if inverse else 0)
    if table is None:
        if positions is not None or axes is not None:
            raise ValueError("positions and axes need a table")
        return (0, 0, 0, 0, None), 0, flags
    _check("table", table, 3, (torch.float32,), device)
    if table.shape[2] != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous [positions, pairs, 2]")
    r = 2 * table.shape[1]
    if r > d:
        raise ValueError(f"the table turns {r} values of head vectors of {d}")
    ax = None
    if axes is not None:
        if len(axes) != 3:
            raise ValueError("axes: the pairs of three axes")
        ax = _Three(*axes)
    if positions is None:
        if start < 0 or start + l > table.shape[0]:
            raise ValueError(f"positions {start}..{start + l - 1} run past the table's {table.shape[0]}")
        return (table.shape[0], 0, 0, int(start), ax), r, flags
    if start:
        raise ValueError("start is for calls without positions")
    shape = positions.shape
    tail = (l,) if ax is None else (l, 3)
    if tuple(shape) == tail:
        batch = 0
    elif tuple(shape) == (b, *tail):
        batch = math.prod(tail) if b > 1 else 0
    else:
        raise ValueError(f"positions must be {tail} or {(b, *tail)}, got {tuple(shape)}")
    _check("positions", positions, len(shape), _POSITION_TYPES, device)
    if not positions.is_contiguous():
        raise ValueError("positions must be contiguous")
    return (table.shape[0], int(positions.dtype == torch.int64), batch, 0, ax), r, flags


_rope_plans: dict = {}
_norm_plans: dict = {}


def _rope_plan(x, table, positions, interleaved, axes, inverse, start, out):
    _check("x", x, 4, DTYPES)
    if table is None:
        raise ValueError("table is required")
    b, l, h, d = x.shape
    dev = x.device
    (rows, p64, batch, first, ax), r, flags = _turns(table, positions, axes, b, l, d, interleaved, inverse, start, dev)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _check_out("out", out, x.shape, x.dtype, dev)
    strides = _Six(*_strides(x, (0, 1, 2)), *_strides(out, (0, 1, 2)))
    return (x.numel() == 0, dev.index, DTYPES[x.dtype], rows, (p64, batch, first, ax, b, l, h, d, r, flags, strides))


def rope(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor | None = None, *, interleaved: bool = True,
         axes=None, inverse: bool = False, start: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns the pairs of ``x`` ``[B,L,H,D]`` (bf16, fp16 or fp32) by the
    positions of its tokens; returns ``[B,L,H,D]``.

    ``table`` ``[positions, R/2, 2]`` (:func:`rope_table`) turns the first R
    of the D values, the rest pass through: pairs ``(2j, 2j+1)`` when
    ``interleaved``, else ``(j, j + R/2)``.  ``positions``: int32 or int64
    ``[L]`` or ``[B,L]``, or ``[.., 3]`` with ``axes`` (the pairs of each
    axis); without them token t is at ``start + t``.  ``inverse`` turns back
    (by the negative angle).  ``out`` may be ``x``; other overlaps are not
    allowed.  A position that is no row of the table gives zeros and sets the
    device error word (:func:`cast_b200._lib.check_device`).
    """
    axes = None if axes is None else tuple(map(int, axes))
    interleaved, inverse, start = bool(interleaved), bool(inverse), int(start)
    try:
        key = (x.dtype, x.shape, x.stride(), x.device, table.dtype, table.shape, table.stride(), table.device,
               None if positions is None else (positions.dtype, positions.shape, positions.stride(), positions.device),
               None if out is None else _sig(out), interleaved, axes, inverse, start)
        plan = _rope_plans.get(key)
    except AttributeError:
        key = plan = None  # (not a tensor: the checks say so)
    if plan is None:
        plan = _keep(_rope_plans, key, _rope_plan(x, table, positions, interleaved, axes, inverse, start, out))
    empty, index, dtype, rows, rest = plan
    _refuse_gradients(x, table, out)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if not empty:
        _launch(index, "cast_rope", x.data_ptr(), dtype, table.data_ptr(), rows,
                None if positions is None else positions.data_ptr(), *rest, out.data_ptr())
    return out


def _norm_plan(q, k, q_weight, k_weight, table, positions, interleaved, axes, start, out_dtype, qo, ko, v, cache, slots):
    _check("q", q, 4, DTYPES)
    dev, dtype = q.device, q.dtype
    _check("k", k, 4, (dtype,), dev)
    b, l, hq, d = q.shape
    hk = k.shape[2]
    if k.shape != (b, l, hk, d):
        raise ValueError(f"k shape {tuple(k.shape)} incompatible with q {tuple(q.shape)}")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype not in DTYPES or (out_dtype != dtype and (dtype, out_dtype) != (torch.float32, torch.bfloat16)):
        raise ValueError("out_dtype: the inputs' type, or bfloat16 of float32 inputs")
    f32 = per_head = None
    for name, w, h in (("q_weight", q_weight, hq), ("k_weight", k_weight, hk)):
        if w is None:
            continue
        _check(name, w, w.ndim, (dtype, torch.float32), dev)
        if tuple(w.shape) not in ((d,), (h, d)) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [D] or [H,D], got {tuple(w.shape)}")
        if f32 not in (None, w.dtype == torch.float32) or per_head not in (None, w.ndim == 2):
            raise ValueError("q_weight and k_weight must have the same type and rank")
        f32, per_head = w.dtype == torch.float32, w.ndim == 2
    (rows, p64, batch, first, ax), r, flags = _turns(table, positions, axes, b, l, d, interleaved, False, start, dev)
    if qo is not None:
        _check_out("out[0]", qo, (b, hq, l, d), out_dtype, dev)
    pages, page, slots64 = 0, 0, 0
    if cache is not None:
        if v is None or slots is None:
            raise ValueError("a cache needs v and slots")
        if ko is not None:
            raise ValueError("the keys go to the cache: out is (q, None)")
        _check("v", v, 4, (dtype,), dev)
        if v.shape != k.shape:
            raise ValueError(f"v shape {tuple(v.shape)} differs from k {tuple(k.shape)}")
        kp, vp = cache
        for name, t in (("k_pages", kp), ("v_pages", vp)):
            _check(name, t, 4, (out_dtype,), dev)
            if t.shape[1] != hk or t.shape[3] != d or t.shape != kp.shape or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [n_pages,{hk},page,{d}], got {tuple(t.shape)}")
        pages, page = kp.shape[0], kp.shape[2]
        _check("slots", slots, 2, _POSITION_TYPES, dev)
        if tuple(slots.shape) != (b, l) or not slots.is_contiguous():
            raise ValueError(f"slots must be a contiguous {(b, l)}, got {tuple(slots.shape)}")
        slots64 = int(slots.dtype == torch.int64)
    elif v is not None or slots is not None:
        raise ValueError("v and slots go with a cache")
    elif ko is not None:
        _check_out("out[1]", ko, (b, hk, l, d), out_dtype, dev)
    empty = b * l == 0
    if not empty and (hq == 0 or hk == 0 or d == 0 or (cache is not None and pages * page == 0)):
        raise ValueError("no heads, or an empty cache")
    strides = _Fifteen(*_strides(q, (0, 1, 2)), *_strides(k, (0, 1, 2)),
                       *(_strides(v, (0, 1, 2)) if cache is not None else (0, 0, 0)),
                       *((hq * l * d, d, l * d) if qo is None else _strides(qo, (0, 2, 1))),
                       *((hk * l * d, d, l * d) if ko is None else _strides(ko, (0, 2, 1))))
    return (empty, dev.index, out_dtype, (b, hq, l, d), (b, hk, l, d), (DTYPES[dtype], DTYPES[out_dtype]),
            (int(bool(f32)), int(bool(per_head))), rows,
            (p64, batch, first, ax, b, l, hq, hk, d, r, flags, strides), (slots64, pages, page))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 table: torch.Tensor | None = None, positions: torch.Tensor | None = None, *, eps: float = 1e-6,
                 interleaved: bool = True, axes=None, start: int = 0, out_dtype: torch.dtype | None = None, out=None,
                 v: torch.Tensor | None = None, cache=None, slots: torch.Tensor | None = None):
    """RMS norm of each head of ``q`` ``[B,L,Hq,D]`` and ``k`` ``[B,L,Hk,D]``
    (``x / sqrt(mean(x^2) + eps) * weight``), then the rotation of
    :func:`rope`, in float32 with one rounding at the end.

    Returns ``(q [B,Hq,L,D], k [B,Hk,L,D])``, the layout the attention takes
    (``out``: a pair of such tensors to write instead, strides free).  The
    inputs may be slices of one projection.  Weights are ``[D]`` or ``[H,D]``,
    of the input type or float32; ``None`` leaves that tensor without a norm,
    ``table=None`` leaves out the rotation.  ``out_dtype``: bf16 of fp32
    inputs.

    With ``cache = (k_pages, v_pages)`` ``[n_pages,Hk,page,D]``, ``v``
    ``[B,L,Hk,D]`` and ``slots`` (int32 or int64 ``[B,L]``), token (b, l)'s
    key and value are written to row ``slots % page`` of page ``slots //
    page`` and the pages are returned in place of k.  A slot below zero is not
    written; one past the end is not written and sets the device error word.
    Slots must differ from one another.
    """
    axes = None if axes is None else tuple(map(int, axes))
    interleaved, start = bool(interleaved), int(start)
    qo, ko = (None, None) if out is None else out
    kp, vp = (None, None) if cache is None else cache
    try:
        key = (q.dtype, q.shape, q.stride(), q.device, k.dtype, k.shape, k.stride(), k.device,
               None if q_weight is None else (q_weight.dtype, q_weight.shape, q_weight.stride(), q_weight.device),
               None if k_weight is None else (k_weight.dtype, k_weight.shape, k_weight.stride(), k_weight.device),
               None if table is None else (table.dtype, table.shape, table.stride(), table.device),
               None if positions is None else (positions.dtype, positions.shape, positions.stride(), positions.device),
               None if out is None else (_sig(qo), _sig(ko)),
               None if cache is v is slots is None else
               (v.dtype, v.shape, v.stride(), v.device, kp.dtype, kp.shape, kp.stride(), kp.device, vp.dtype, vp.shape,
                vp.stride(), vp.device, slots.dtype, slots.shape, slots.stride(), slots.device),
               interleaved, axes, start, out_dtype)
        plan = _norm_plans.get(key)
    except AttributeError:
        key = plan = None  # (not a tensor: the checks say so)
    if plan is None:
        plan = _keep(_norm_plans, key, _norm_plan(q, k, q_weight, k_weight, table, positions, interleaved, axes, start,
                                                  out_dtype, qo, ko, v, cache, slots))
    empty, index, out_dtype, q_shape, k_shape, types, weights, rows, rest, places = plan
    _refuse_gradients(q, k, q_weight, k_weight, table, v, kp, vp, qo, ko)
    if qo is None:
        qo = q.new_empty(q_shape) if out_dtype is q.dtype else q.new_empty(q_shape, dtype=out_dtype)
    if cache is None and ko is None:
        ko = q.new_empty(k_shape) if out_dtype is q.dtype else q.new_empty(k_shape, dtype=out_dtype)
    if not empty:
        P = _lib.ptr
        _launch(index, "cast_qk_norm_rope", q.data_ptr(), k.data_ptr(), P(v), *types, P(q_weight), P(k_weight), *weights,
                eps, P(table), rows, P(positions), *rest, qo.data_ptr(), (ko if cache is None else kp).data_ptr(), P(vp), P(slots),
                *places)
    return (qo, ko) if cache is None else (qo, cache)
