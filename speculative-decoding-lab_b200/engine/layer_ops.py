"""Fused elementwise ops of a decoder layer for 16-bit models on CUDA.

``rmsnorm`` / ``add_rmsnorm`` / ``rope_`` / ``silu_mul`` each replace a chain
of small framework kernels of engine/model.py and engine/qwen.py with one
launch of ``csrc/layer_ops.cu`` and round where the chain rounds (RMSNorm's
mean may differ in the last fp32 bit: its sum order is the kernel's).
``fusable(x)`` says whether a tensor takes this path; fp32 models keep the
framework ops.

``rope_axes`` (``csrc/rotary.cu``) is not one of those chains: it rotates q
and k of any supported dtype straight from a position table, with a position
per axis (time, height, width), in fp32 with one rounding.
"""

from __future__ import annotations

import ctypes
import threading
from typing import Optional, Sequence, Tuple

import torch

from . import _lib


def fusable(x: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype in (torch.bfloat16, torch.float16)


def _rows(x: torch.Tensor) -> torch.Tensor:
    x2 = x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(-1) == 1 else x2.contiguous()


def add_rmsnorm(x: torch.Tensor, delta, weight: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + delta`` (when ``delta`` is given) and ``rmsnorm(h)``; returns ``(h, normed)``."""
    xr = _rows(x)
    out = torch.empty(xr.shape, dtype=x.dtype, device=x.device)
    if delta is not None:
        dr = _rows(delta)
        h = torch.empty_like(out)
        args = (dr.data_ptr(), dr.stride(0), h.data_ptr(), h.stride(0))
    else:
        h = None
        args = (None, 0, None, 0)
    w = weight if weight.dtype == x.dtype else weight.to(x.dtype)
    _lib.check(
        _lib.load().sdl_rmsnorm(xr.data_ptr(), xr.stride(0), *args, w.data_ptr(), out.data_ptr(), out.stride(0),
                                xr.shape[0], xr.shape[1], float(eps), _lib.dtype_code(x.dtype),
                                _lib.stream_handle(x.device)),
        "sdl_rmsnorm",
    )
    normed = out.reshape(x.shape)
    return (h.reshape(x.shape) if h is not None else x), normed


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return add_rmsnorm(x, None, weight, eps)[1]


def rope_(x: torch.Tensor, sin: torch.Tensor, cos: torch.Tensor) -> torch.Tensor:
    """In-place ``x * cos + rotate_half(x) * sin`` for ``x`` of shape
    ``(..., heads, d)`` with contiguous rows; ``cos`` / ``sin`` hold one
    ``d``-row per leading position of ``x`` (broadcast over heads)."""
    d = x.shape[-1]
    heads = x.shape[-2]
    xr = x.reshape(-1, heads * d)
    if xr.stride(-1) != 1 or (xr.data_ptr() != x.data_ptr()):
        raise ValueError("rope_: rows of x must be contiguous")
    c = cos.reshape(-1, d)
    s = sin.reshape(-1, d)
    if c.shape[0] != xr.shape[0] or s.shape[0] != xr.shape[0] or c.stride(-1) != 1 or s.stride(-1) != 1:
        raise ValueError("rope_: cos/sin must hold one row per position of x")
    c = c if c.dtype == x.dtype else c.to(x.dtype)
    s = s if s.dtype == x.dtype else s.to(x.dtype)
    _lib.check(
        _lib.load().sdl_rope(xr.data_ptr(), xr.stride(0), xr.shape[0], heads, d, c.data_ptr(), c.stride(0),
                             s.data_ptr(), s.stride(0), _lib.dtype_code(x.dtype), _lib.stream_handle(x.device)),
        "sdl_rope",
    )
    return x


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` with the framework's two roundings."""
    g = gate.contiguous()
    u = up.contiguous()
    out = torch.empty_like(g)
    _lib.check(
        _lib.load().sdl_silu_mul(g.data_ptr(), u.data_ptr(), out.data_ptr(), g.numel(), _lib.dtype_code(g.dtype),
                                 _lib.stream_handle(g.device)),
        "sdl_silu_mul",
    )
    return out


def swiglu(gate_up: torch.Tensor, inter: int) -> torch.Tensor:
    """``silu(gate) * up`` on rows ``[gate | up]`` of one fused projection
    (``inter`` columns each), with ``silu_mul``'s two roundings."""
    x = gate_up.reshape(-1, gate_up.shape[-1])
    if x.stride(-1) != 1:
        x = x.contiguous()
    out = torch.empty((x.shape[0], inter), dtype=x.dtype, device=x.device)
    _lib.check(
        _lib.load().sdl_swiglu(x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), x.shape[0], int(inter),
                               _lib.dtype_code(x.dtype), _lib.stream_handle(x.device)),
        "sdl_swiglu",
    )
    return out.reshape(*gate_up.shape[:-1], inter)



def _rope_args(table: torch.Tensor, positions: torch.Tensor, sections: Optional[Sequence[int]], tokens: int,
               head_dim: int, device: torch.device) -> _lib.SdlRopeArgs:
    """Checked table, position and section fields of a rotation's arguments
    (all but the pointers, which change from call to call)."""
    if table.dim() != 3 or table.shape[1] != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table must be contiguous float32 (max_len, 2, rotary), as make_rotary_cache returns")
    rotary = table.shape[2]
    if rotary < 2 or rotary % 2 or rotary > head_dim or table.shape[0] < 1:
        raise ValueError("table: rotary width {} must be even and at most head_dim {}".format(rotary, head_dim))
    if tokens > ROPE_TOKENS_MAX:
        raise ValueError("{} rows in one call, of {} at most".format(tokens, ROPE_TOKENS_MAX))
    nd = positions.dim()
    if nd not in (1, 2) or positions.shape[-1] != tokens:
        raise ValueError("positions must be (tokens,) or (axes, tokens) for {} tokens, got {}".format(
            tokens, tuple(positions.shape)))
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError("positions must be int64 or int32, got {}".format(positions.dtype))
    if table.device != device or positions.device != device:
        raise ValueError("table and positions must be on {}".format(device))
    axes = 1 if nd == 1 else positions.shape[0]
    if not 1 <= axes <= 4:
        raise ValueError("positions of one to four axes are supported, got {}".format(axes))
    if sections is None:
        if axes != 1:
            raise ValueError("positions of {} axes need their sections".format(axes))
        sections = (rotary // 2,)
    if len(sections) != axes or min(sections) < 0 or sum(sections) * 2 != rotary:
        raise ValueError("sections must give each of {} axes its pairs, {} in all, got {}".format(
            axes, rotary // 2, tuple(sections)))
    a = _lib.SdlRopeArgs()
    a.table_rows, a.rotary, a.axes = table.shape[0], rotary, axes
    a.pos64 = 1 if positions.dtype == torch.int64 else 0
    a.pos_stride = positions.stride(0) if axes > 1 else 0
    for i, n in enumerate(sections):
        a.sections[i] = int(n)
    a.num_tokens, a.head_dim = tokens, head_dim
    return a


def _check_heads(x: torch.Tensor, name: str, tokens: int, heads: Optional[int], head_dim: int, dtype: torch.dtype,
                 device: torch.device) -> None:
    want = (tokens, x.shape[1] if heads is None and x.dim() == 3 else heads, head_dim)
    if tuple(x.shape) != want or x.dtype != dtype or x.device != device:
        raise ValueError("{} must be (tokens, heads, head_dim) = {} of {} on {}, got {} of {} on {}".format(
            name, want, dtype, device, tuple(x.shape), x.dtype, x.device))


def _has_head_rows(x: torch.Tensor) -> bool:
    """Unit-stride, back-to-back heads (rows may be strided).  A tensor without
    elements has them whatever its strides, which a copy would keep."""
    return x.numel() == 0 or (
        (x.stride(2) == 1 or x.shape[2] == 1) and (x.stride(1) == x.shape[2] or x.shape[1] == 1))


def _check_out_rows(x: torch.Tensor, name: str) -> None:
    if not _has_head_rows(x) or (x.shape[0] > 1 and x.stride(0) < x.shape[1] * x.shape[2]):
        raise ValueError("{} needs rows of back-to-back heads that do not overlap".format(name))


def check_apart(plan: "RopePlan", outs, inputs) -> None:
    """Refuses outputs that share memory with each other or with an input;
    ``outs`` are (name, output) in the order of their inputs, and an output may
    be its own input itself.  The answer holds for the tensors' distances and row strides."""
    base = inputs[0].data_ptr()
    sig = tuple(t.data_ptr() - base for t in inputs) + tuple(
        x for _, o in outs for x in (o.data_ptr() - base, o.stride(0)))
    if sig == plan.apart:
        return
    for i, (name, o) in enumerate(outs):
        for j, t in enumerate(inputs):
            if not (j == i and _lib.same_elements(o, t)) and _lib.share_memory(o, t):
                raise ValueError("{} must be its input itself or not overlap any".format(name))
        for _, other in outs[:i]:
            if _lib.share_memory(o, other):
                raise ValueError("{} must not overlap another output".format(name))
    plan.apart = sig


def _empty_contiguous(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


class RopePlan:
    """A checked argument struct of one combination of shapes, strides, types
    and thread; calls that hit it fill in the pointers."""

    __slots__ = ("args", "ref", "device", "like_q", "like_k", "apart")

    def __init__(self, args: _lib.SdlRopeArgs, device: torch.device, q: Optional[torch.Tensor],
                 k: Optional[torch.Tensor]) -> None:
        self.args = args
        self.ref = ctypes.byref(args)
        self.device = device
        self.apart = None  # distances of the tensors that check_apart has passed
        # new outputs (a contiguous input's layout is the default, which takes 0.3 us less)
        self.like_q, self.like_k = (
            torch.empty_like if x is None or x.is_contiguous() else _empty_contiguous for x in (q, k))

    def launch(self, fn: str) -> None:
        dev = self.device
        if _lib.current_device() == dev.index:
            rc = getattr(_lib.load(), fn)(self.ref, _lib.stream_handle(dev))
        else:  # a launch needs its stream's device current
            with torch.cuda.device(dev):
                rc = getattr(_lib.load(), fn)(self.ref, _lib.stream_handle(dev))
        _lib.check(rc, fn)


_ROPE_PLANS = {}
ROPE_PLANS_MAX = 256
ROPE_TOKENS_MAX = 2 ** 31 - 65  # rows are counted in 32 bits, a block's 64 past the last included


def rope_key(q, k, table, positions, sections):
    """What a ``RopePlan`` depends on."""
    return (q.shape, q.stride(), q.dtype, q.get_device(),
            None if k is None else (k.shape, k.stride(), k.dtype, k.get_device()),
            table.shape, table.stride(), table.dtype, table.get_device(),
            positions.shape, positions.stride(), positions.dtype, positions.get_device(),
            None if sections is None else tuple(sections), threading.get_ident())


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: torch.Tensor,
              sections: Optional[Sequence[int]] = None,
              out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None):
    """Rotate-half RoPE of ``q (T, Hq, d)`` and ``k (T, Hkv, d)`` (or None)
    by positions of one or several axes; returns the turned ``(q, k)``.

    ``table`` is ``make_rotary_cache``'s ``(max_len, 2, R)`` fp32 cos / sin
    table, ``R <= d`` (dims past ``R`` are copied).  ``positions`` is ``(T,)``,
    or ``(axes, T)`` with ``sections`` giving how many of the ``R/2`` pairs
    each axis turns, in order: pair ``i`` (dims ``i`` and ``i + R/2``) of row
    ``t`` turns by ``table[positions[axis of i, t], :, i]``.  The arithmetic
    is fp32, rounded once (``rope_`` keeps the framework chain's roundings
    instead).  A pair whose position lies outside the table comes out NaN, the
    row's other pairs as usual.

    ``out = (q_out, k_out)`` receives the result (rows of back-to-back heads).
    They may be ``q`` and ``k`` themselves, each its own input; outputs that
    overlap an input otherwise, or each other, are refused.
    """
    key = rope_key(q, k, table, positions, sections)
    plan = _ROPE_PLANS.get(key)
    if plan is None:
        _lib.require_cuda(q, "q")
        if q.dim() != 3:
            raise ValueError("q must be (tokens, heads, head_dim), got {}".format(tuple(q.shape)))
        T, hq, d = q.shape
        if k is not None:
            _check_heads(k, "k", T, None, d, q.dtype, q.device)
        a = _rope_args(table, positions, sections, T, d, q.device)
        a.dtype = _lib.dtype_code(q.dtype)
        if not _has_head_rows(q) or (k is not None and not _has_head_rows(k)) \
                or (T > 1 and positions.stride(-1) != 1):
            return rope_axes(q.contiguous(), None if k is None else k.contiguous(), table, positions.contiguous(),
                             sections, out)
        a.Hq, a.q_row_stride = hq, q.stride(0)
        if k is not None:
            a.Hkv, a.k_row_stride = k.shape[1], k.stride(0)
        if len(_ROPE_PLANS) >= ROPE_PLANS_MAX:
            _ROPE_PLANS.clear()
        plan = RopePlan(a, q.device, q, k)
        _ROPE_PLANS[key] = plan
    a = plan.args
    if out is None:
        qo = plan.like_q(q)
        a.q_out_row_stride = a.Hq * a.head_dim
        ko = None
        if k is not None:
            ko = plan.like_k(k)
            a.k_out_row_stride = a.Hkv * a.head_dim
    else:
        qo, ko = out
        for name, o, x in (("q", qo, q), ("k", ko, k)):
            if (o is None) != (x is None):
                raise ValueError("out must hold what q and k hold")
            if o is not None:
                _check_heads(o, "out: " + name, x.shape[0], x.shape[1], x.shape[2], x.dtype, x.device)
                _check_out_rows(o, "out: " + name)
        if k is None:
            check_apart(plan, (("out: q", qo),), (q,))
        else:
            check_apart(plan, (("out: q", qo), ("out: k", ko)), (q, k))
        a.q_out_row_stride = qo.stride(0)
        a.k_out_row_stride = 0 if ko is None else ko.stride(0)
    if not a.num_tokens or not (a.Hq or a.Hkv):
        return qo, ko
    if a.Hq:
        a.q, a.q_out = q.data_ptr(), qo.data_ptr()
    if a.Hkv:
        a.k, a.k_out = k.data_ptr(), ko.data_ptr()
    a.table, a.positions = table.data_ptr(), positions.data_ptr()
    plan.launch("sdl_rope_axes")
    return qo, ko
