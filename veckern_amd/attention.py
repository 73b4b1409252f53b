"""Attention to the states of what a search found, its position bias by buckets, and their gradients.

Python binding of ``vk_attend`` and ``vk_attend_backward`` (``include/veckern/veckern.h`` states the formulas) for torch
tensors on the GPU. A search returns ids of rows; an encoder's states of those rows, keys and values
``[bank, length, kv_heads, head_dim]``, lie in a bank; ``attend`` lets query tokens attend to the rows a search found for
them, without a copy of what was found:

    ids = records[..., 1]                     # int32 view of the search's (dist, id) records on the device
    out = attend(q, keys, values, rows=ids, lengths=lengths)

Without ``rows`` the bank itself holds each request's rows in order, as an encoder leaves them in training; then
``attend`` takes part in torch's automatic differentiation, or ``attend_backward`` is called with what the forward pass
returned. Work is launched on torch's current stream, and nothing waits for it. There is no CPU form.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch

from . import (VK_ERR_INVALID_ARGUMENT, VkInvalidArgument, _Attention, _AttentionGrad, _check, _Tensor, library)

__all__ = ["RelativeBias", "Gradients", "attend", "attend_backward", "bias_bucket"]

_TYPES = {torch.float16: 0, torch.bfloat16: 1}


@dataclass(frozen=True)
class RelativeBias:
    """A learned bias added to the logits: ``table[bucket(key position - query position), head]``.

    ``table``: ``[buckets, heads]``, of the queries' type. Of a side's buckets (all, or half of them for each direction
    where ``two_sided``) the first half hold one distance each, the others grow by a common factor up to ``max_distance``;
    ``bias_bucket`` gives the bucket of a distance. One-sided, keys after the query share the bucket of distance 0.
    """

    table: torch.Tensor
    max_distance: int = 128
    two_sided: bool = True


class Gradients(NamedTuple):
    """What ``attend_backward`` returns; ``keys`` and ``values`` are None for rows of a bank, ``table`` without a bias."""

    queries: torch.Tensor
    keys: Optional[torch.Tensor]
    values: Optional[torch.Tensor]
    table: Optional[torch.Tensor]


def bias_bucket(distance: int, buckets: int, max_distance: int = 128, two_sided: bool = True) -> int:
    """The bucket of ``distance`` = key position - query position (``vk_bias_bucket``)."""
    b = ctypes.c_int()
    _check(library().vk_bias_bucket(distance, buckets, max_distance, int(two_sided), ctypes.byref(b)))
    return b.value


def _refuse(message: str):
    raise VkInvalidArgument(VK_ERR_INVALID_ARGUMENT, message)


def _view(t: torch.Tensor, name: str, shape: tuple, like: torch.Tensor) -> _Tensor:
    if t.shape != shape or t.dtype != like.dtype or t.device != like.device:
        _refuse(f"{name} must be {list(shape)} {like.dtype} on {like.device}, not {list(t.shape)} {t.dtype} on {t.device}")
    a, b, c, d = t.stride()
    if d != 1:
        _refuse(f"{name}: the elements of a head must be contiguous")
    return _Tensor(t.data_ptr(), (a, b, c))


def _indices(t: torch.Tensor, name: str, shape: tuple, like: torch.Tensor, strided: bool) -> None:
    if t.shape != shape or t.dtype != torch.int32 or t.device != like.device:
        _refuse(f"{name} must be {list(shape)} int32 on {like.device}, not {list(t.shape)} {t.dtype} on {t.device}")
    if not strided and not t.is_contiguous():
        _refuse(f"{name} must be contiguous")


def _arguments(q, keys, values, rows, lengths, bias, q_start, scale) -> _Attention:
    """Everything of a call but its addresses."""
    if not q.is_cuda:
        _refuse("queries must be on a GPU")
    if q.dim() != 4 or keys.dim() != 4:
        _refuse("queries must be [batch, tokens, heads, d] and keys [bank, length, kv_heads, d]")
    kind = _TYPES.get(q.dtype)
    if kind is None:
        _refuse(f"queries must be float16 or bfloat16, not {q.dtype}")
    batch, tokens, heads, d = q.shape
    bank, length, kv_heads, kd = keys.shape
    if kd != d:
        _refuse(f"keys have {kd} elements a head, queries {d}")
    a = _Attention()
    a.type, a.batch, a.tokens, a.heads, a.kv_heads, a.head_dim, a.length, a.bank = (
        kind, batch, tokens, heads, kv_heads, d, length, bank)
    if rows is None:
        if batch == 0 or bank % batch:
            if bank:
                _refuse(f"without rows, the bank's {bank} rows must be a multiple of the batch ({batch})")
            a.passages = 0
        else:
            a.passages = bank // batch
    else:
        if rows.dim() != 2:
            _refuse("rows must be [batch, passages]")
        a.passages = rows.shape[1]
        _indices(rows, "rows", (batch, rows.shape[1]), q, True)
        a.rows = 1  # there are some; the address follows
        a.rows_stride = rows.stride()
    a.scale = 1.0 / math.sqrt(d) if scale is None else scale
    a.q = _view(q, "queries", q.shape, q)
    a.k = _view(keys, "keys", keys.shape, q)
    a.v = _view(values, "values", keys.shape, q)
    if lengths is not None:
        _indices(lengths, "lengths", (bank,), q, False)
    if bias is not None:
        t = bias.table
        if t.dim() != 2 or t.shape[0] == 0 or t.shape[1] != heads or t.dtype != q.dtype or t.device != q.device:
            _refuse(f"the bias table must be [buckets, {heads}] {q.dtype} on {q.device}, not {list(t.shape)} {t.dtype} on "
                    f"{t.device}")
        a.table, a.table_stride, a.buckets = 1, t.stride(), t.shape[0]
        a.max_distance, a.two_sided = bias.max_distance, bias.two_sided
    if isinstance(q_start, torch.Tensor):
        _indices(q_start, "q_start", (batch,), q, False)
    else:
        a.q_start = q_start
    return a


class _Plan:
    """What calls with the same sizes, strides, types and devices share: the arguments but for the addresses."""

    __slots__ = ("image", "forward_bytes", "backward_bytes", "lse_shape", "grads")

    def __init__(self, image, forward_bytes, backward_bytes, lse_shape):
        self.image, self.forward_bytes, self.backward_bytes, self.lse_shape = image, forward_bytes, backward_bytes, lse_shape
        self.grads = {}  # by the kinds of what the backward pass is given besides: the gradients' strides


_plans: dict = {}
_MOST_PLANS = 512


def _kind(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _plan(q, keys, values, rows, lengths, bias, q_start, scale) -> _Plan:
    key = (_kind(q), _kind(keys), _kind(values), _kind(rows), _kind(lengths),
           None if bias is None else (_kind(bias.table), bias.max_distance, bias.two_sided),
           _kind(q_start) if isinstance(q_start, torch.Tensor) else q_start, scale)
    plan = _plans.get(key)
    if plan is None:
        a = _arguments(q, keys, values, rows, lengths, bias, q_start, scale)
        lib, forward, backward = library(), ctypes.c_size_t(), ctypes.c_size_t()
        _check(lib.vk_attend_workspace(ctypes.byref(a), ctypes.byref(forward)))
        _check(lib.vk_attend_backward_workspace(ctypes.byref(a), ctypes.byref(backward)))
        plan = _Plan(bytes(a), forward.value, backward.value, (a.batch, a.heads, a.tokens, 2))
        if len(_plans) >= _MOST_PLANS:
            _plans.clear()
        _plans[key] = plan
    return plan


_ADDRESS = struct.Struct("P")
_AT = {name: getattr(_Attention, name).offset for name in ("q", "k", "v", "out", "rows", "lengths", "lse", "table", "q_starts")}
_GRAD_AT = {name: getattr(_AttentionGrad, name).offset for name in ("d_q", "d_k", "d_v", "d_table")}
_OUT_STRIDE = _AT["out"] + _Tensor.stride.offset
_STRIDES = struct.Struct("3q")


def _contiguous(shape) -> tuple:
    _, b, c, d = shape
    return (b * c * d, c * d, d)


def _filled(plan, q, keys, values, out, lse, rows, lengths, bias, q_start) -> _Attention:
    a, put = bytearray(plan.image), _ADDRESS.pack_into
    put(a, _AT["q"], q.data_ptr())
    put(a, _AT["k"], keys.data_ptr())
    put(a, _AT["v"], values.data_ptr())
    put(a, _AT["out"], out.data_ptr())
    _STRIDES.pack_into(a, _OUT_STRIDE, *out.stride()[:3])
    if rows is not None:
        put(a, _AT["rows"], rows.data_ptr() or 1)  # without elements: any address, there is nothing to read
    if lengths is not None:
        put(a, _AT["lengths"], lengths.data_ptr())
    if lse is not None:
        put(a, _AT["lse"], lse.data_ptr())
    if bias is not None:
        put(a, _AT["table"], bias.table.data_ptr())
    if isinstance(q_start, torch.Tensor):
        put(a, _AT["q_starts"], q_start.data_ptr())
    return _Attention.from_buffer(a)


def _launch(entry, arguments, size, device):
    """Calls ``entry(*arguments, workspace, bytes, stream)`` on the device's current stream."""
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    at = work.data_ptr() if size else None
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = entry(*arguments, at, size, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*arguments, at, size, stream)
    if rc:
        _check(rc)


def _forward(q, keys, values, rows, lengths, bias, q_start, scale, with_lse):
    plan = _plan(q, keys, values, rows, lengths, bias, q_start, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(plan.lse_shape, dtype=torch.float32, device=q.device) if with_lse else None
    a = _filled(plan, q, keys, values, out, lse, rows, lengths, bias, q_start)
    _launch(library().vk_attend, (a,), plan.forward_bytes, q.device)
    return out, lse


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, keys, values, table, rows, lengths, bias, q_start, scale):
        out, lse = _forward(q, keys, values, rows, lengths, bias, q_start, scale, True)
        starts = q_start if isinstance(q_start, torch.Tensor) else None
        ctx.save_for_backward(q, keys, values, table, rows, lengths, starts, out, lse)
        ctx.rest = (None if bias is None else (bias.max_distance, bias.two_sided), q_start if starts is None else None, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, d_out, _):
        q, keys, values, table, rows, lengths, starts, out, lse = ctx.saved_tensors
        kind, q_start, scale = ctx.rest
        bias = None if kind is None else RelativeBias(table, *kind)
        # the chain may hand over any strides (a sum's gradient is one element, repeated)
        g = attend_backward(d_out.contiguous(), q, keys, values, out, lse, rows=rows, lengths=lengths, bias=bias,
                            q_start=q_start if starts is None else starts, scale=scale)
        return (*g, None, None, None, None, None)


def attend(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, *, rows: Optional[torch.Tensor] = None,
           lengths: Optional[torch.Tensor] = None, bias: Optional[RelativeBias] = None, q_start=0,
           scale: Optional[float] = None, return_lse: bool = False):
    """Attention of ``q`` ``[batch, tokens, heads, d]`` to the states of each request's rows; returns ``out`` of q's shape.

    ``keys``, ``values``: ``[bank, length, kv_heads, d]`` (float16 or bfloat16 as ``q``; d a multiple of 8, at most 128;
    ``heads`` a multiple of ``kv_heads``). ``rows``: int32 ``[batch, passages]`` ids of bank rows, any strides; ids outside
    the bank (a search's -1) hold nothing. Without it request b has the rows ``b * passages ...`` of a bank of
    ``batch * passages``. ``lengths``: int32 ``[bank]``, positions that a row holds (all where not given). ``q_start``: the
    position of token 0, a number or int32 ``[batch]``; it matters to ``bias`` alone. ``scale``: by default
    ``1 / sqrt(d)``. ``return_lse``: also returns the logarithm of each row's sum of exponentials, float32
    ``[batch, heads, tokens, 2]``: its value and what rounding that to 32 bits left off. A token with nothing to attend to gets zeros (lse: -inf).

    Gradients flow to ``q``, ``keys``, ``values`` and ``bias.table``, except to a bank that is read by ``rows``: it counts
    as a constant, and one that requires a gradient is refused.
    """
    table = None if bias is None else bias.table
    if torch.is_grad_enabled() and (q.requires_grad or keys.requires_grad or values.requires_grad
                                    or (table is not None and table.requires_grad)):
        if rows is not None and (keys.requires_grad or values.requires_grad):
            _refuse("a bank that is read by rows has no gradient: detach it, or select its rows first")
        out, lse = _Attend.apply(q, keys, values, table, rows, lengths, bias, q_start, scale)
    else:
        out, lse = _forward(q, keys, values, rows, lengths, bias, q_start, scale, return_lse)
    return (out, lse) if return_lse else out


def attend_backward(d_out: torch.Tensor, q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, out: torch.Tensor,
                    lse: torch.Tensor, *, rows: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                    bias: Optional[RelativeBias] = None, q_start=0, scale: Optional[float] = None) -> Gradients:
    """The gradients of a loss whose gradient by ``out`` is ``d_out``; ``out`` and ``lse`` as ``attend`` returned them for
    the same arguments. With ``rows`` the bank is a constant and has none."""
    plan = _plan(q, keys, values, rows, lengths, bias, q_start, scale)
    kind = (_kind(d_out), _kind(out), _kind(lse))
    grads = plan.grads.get(kind)
    if grads is None:
        if lse.shape != plan.lse_shape or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
            _refuse(f"lse must be contiguous {list(plan.lse_shape)} float32 on {q.device}")
        _view(out, "out", q.shape, q)
        g = _AttentionGrad()
        g.d_out = _view(d_out, "d_out", q.shape, q)
        g.d_q.stride = _contiguous(q.shape)
        g.d_k.stride = g.d_v.stride = _contiguous(keys.shape)
        if len(plan.grads) >= _MOST_PLANS:
            plan.grads.clear()
        grads = plan.grads[kind] = bytes(g)
    a = _filled(plan, q, keys, values, out, lse, rows, lengths, bias, q_start)
    g, put = bytearray(grads), _ADDRESS.pack_into
    d_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    d_k = d_v = d_table = None
    put(g, 0, d_out.data_ptr())
    put(g, _GRAD_AT["d_q"], d_q.data_ptr())
    if rows is None:
        d_k = torch.empty(keys.shape, dtype=q.dtype, device=q.device)
        d_v = torch.empty(keys.shape, dtype=q.dtype, device=q.device)
        put(g, _GRAD_AT["d_k"], d_k.data_ptr())
        put(g, _GRAD_AT["d_v"], d_v.data_ptr())
    if bias is not None:
        d_table = torch.empty(bias.table.shape, dtype=q.dtype, device=q.device)
        put(g, _GRAD_AT["d_table"], d_table.data_ptr())
    _launch(library().vk_attend_backward, (a, _AttentionGrad.from_buffer(g)), plan.backward_bytes, q.device)
    return Gradients(d_q, d_k, d_v, d_table)
