"""Rotary positions with several axes, with their gradient: tokens of images and video have a time, a row and a column, and every
pair of columns of a head is turned by the position on its own axis. One kernel of the library (``fsa_rotary_axes``) for both
tensors and both directions, beside the single axis of ``rotary.py``; the reference leaves this step to its caller."""

import ctypes
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from flash_sparse_attn import _lib
from flash_sparse_attn.ops.triton.rotary import _rows, _strides, _unseen, check_tables

_F16 = (torch.float16, torch.bfloat16)


def axis_bits(sections: Tuple[int, ...], pairs: int, dealt: bool) -> bytes:
    """The axis of every pair, two bits each (eight words), for ``sections[a]`` pairs of axis a: run after run, or dealt out in turn."""
    return _axis_bits(pairs, dealt, *sections)


@lru_cache(maxsize=256, typed=True)  # (each number by itself: 16.0 is not taken for the 16 of an earlier call)
def _axis_bits(pairs, dealt, *sections):
    assert 2 <= len(sections) <= _lib.MAX_AXES, f"sections must name two to {_lib.MAX_AXES} axes"
    assert all(type(n) is int and n > 0 for n in sections) and sum(sections) == pairs, "sections must be positive and add up to rotary_dim / 2"
    assert pairs <= 128, "rotary_dim must be less than or equal to 256"
    axes, word = len(sections), 0
    if dealt:
        assert all(a + axes * (n - 1) < pairs for a, n in enumerate(sections) if a), "sections do not fit when they are dealt out in turn"
        owner = [i % axes if i // axes < sections[i % axes] else 0 for i in range(pairs)]
    else:
        owner = [a for a, n in enumerate(sections) for _ in range(n)]
    for i, a in enumerate(owner):
        word |= a << (2 * i)
    return word.to_bytes(32, "little")


def check_positions(position_ids, sections, tokens, device):
    """The contract of positions on several axes, shared with ``append_kv_quantized``. ``tokens``: the leading sizes of the rows."""
    assert isinstance(position_ids, torch.Tensor) and position_ids.dtype in (torch.int32, torch.int64), "position_ids must be int32 or int64"
    assert position_ids.device == device, "All inputs must be on the same device"
    shared = (1,) + tuple(tokens[1:]) if len(tokens) == 2 else tuple(tokens)  # one row of positions for the whole batch
    assert tuple(position_ids.shape) in ((len(sections),) + tuple(tokens), (len(sections),) + shared), (
        "position_ids must have one entry per axis and token")


def position_strides(position_ids):
    """(axis, batch, token) strides; a batch that shares its positions has none."""
    if position_ids.ndim == 2:
        return position_ids.stride(0), 0, position_ids.stride(1)
    return position_ids.stride(0), position_ids.stride(1) if position_ids.shape[1] > 1 else 0, position_ids.stride(2)


def _check(query, key, cos, sin, position_ids, sections):
    assert query.ndim in (3, 4), "query must be [batch, seqlen, heads, head_dim] or packed [tokens, heads, head_dim]"
    assert query.dtype in _F16, "Input dtype must be float16 or bfloat16"
    assert query.shape[-1] <= 256, "head_dim must be less than or equal to 256"
    if key is not None:
        assert key.dtype == query.dtype, "All inputs must have the same dtype"
        assert key.ndim == query.ndim and key.shape[:-2] == query.shape[:-2] and key.shape[-1] == query.shape[-1], (
            "query and key must agree in their tokens and head_dim")
        assert key.device == query.device, "All inputs must be on the same device"
    check_tables(cos, sin, query.shape[-1], query.device)
    check_positions(position_ids, sections, query.shape[:-2], query.device)


def _launch(query, key, cos, sin, position_ids, bits, axes, interleaved, transposed):
    device = query.device
    query, key = _rows(query), _rows(key)
    q_out = torch.empty(query.shape, dtype=query.dtype, device=device)
    k_out = None if key is None else torch.empty(key.shape, dtype=key.dtype, device=device)
    if not q_out.numel() and (k_out is None or not k_out.numel()):
        return q_out, k_out
    a = _lib.FsaRotaryAxesArgs()
    a.q, a.q_out, a.cos, a.sin = query.data_ptr(), q_out.data_ptr(), cos.data_ptr(), sin.data_ptr()
    a.k, a.k_out = _lib.ptr(key), _lib.ptr(k_out)
    a.position_ids, a.position_ids_int64 = position_ids.data_ptr(), int(position_ids.dtype == torch.int64)
    a.position_stride_a, a.position_stride_b, a.position_stride_s = position_strides(position_ids)
    a.status = _lib.status_word(device).data_ptr()
    a.q_stride_b, a.q_stride_s, a.q_stride_h = _strides(query)
    a.q_out_stride_b, a.q_out_stride_s, a.q_out_stride_h = _strides(q_out)
    if key is not None:
        a.k_stride_b, a.k_stride_s, a.k_stride_h = _strides(key)
        a.k_out_stride_b, a.k_out_stride_s, a.k_out_stride_h = _strides(k_out)
    a.batch, a.seqlen = query.shape[:2] if query.ndim == 4 else (1, query.shape[0])
    a.heads_q, a.head_dim = query.shape[-2:]
    a.heads_k = 0 if key is None else key.shape[-2]
    a.table_rows, a.rotary_dim, a.table_stride = cos.shape[0], 2 * cos.shape[1], cos.stride(0)
    ctypes.memmove(a.axis_bits, bits, 32)
    a.axes = axes
    a.dtype, a.table_dtype = _lib.dtype_code(query.dtype), _lib.dtype_code(cos.dtype)
    a.interleaved, a.transposed = int(interleaved), int(transposed)
    with torch.cuda.device(device):
        rc = _lib.load().fsa_rotary_axes(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_rotary_axes")
    return q_out, k_out


class _RotaryAxes(torch.autograd.Function):
    """The rotation with its gradient: the transposed rotation of the gradients, which is a rotation again and has a gradient too."""

    @staticmethod
    def forward(ctx, query, key, cos, sin, position_ids, bits, axes, interleaved, transposed):
        ctx.save_for_backward(cos, sin, position_ids)
        ctx.how = bits, axes, interleaved, not transposed
        ctx.set_materialize_grads(False)
        return _launch(query, key, cos, sin, position_ids, bits, axes, interleaved, transposed)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, position_ids = ctx.saved_tensors
        dq, dk = (g if needed else None for g, needed in zip((dq, dk), ctx.needs_input_grad))
        how = (cos, sin, position_ids) + ctx.how
        if dq is not None:
            dq, dk = _turn(dq, dk, *how)
        elif dk is not None:  # a launch's first tensor is the one that is there
            dk = _turn(dk, None, *how)[0]
        return (dq, dk) + (None,) * 7


def _turn(query, key, *how):
    if not _unseen() or (torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))):
        return _RotaryAxes.apply(query, key, *how)
    return _launch(query, key, *how)


def apply_rotary_axes_func(
    query: torch.Tensor,
    key: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    position_ids: torch.Tensor,
    sections: Sequence[int],
    axes_dealt: bool = False,
    interleaved: bool = False,
    skip_checks: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``apply_rotary_func`` for tokens with a position on each of two to four axes (time, height, width): pair ``i`` of a head is turned
    by ``cos / sin[position_ids[a, token], i]`` (tables ``[positions, R / 2]``, fp32 or 16 bits), ``a`` being the pair's axis. ``sections``
    says how many of the ``R / 2`` pairs each axis has: the first ``sections[0]`` are the first axis's, and so on, or with ``axes_dealt``
    pair ``i`` belongs to axis ``i mod len(sections)`` while that axis has pairs left, and to the first one after that.

    ``query [B, S, Hq, D]`` and ``key [B, S, Hkv, D]`` (or None) take ``position_ids [axes, B, S]`` (``[axes, 1, S]`` where the batch shares
    them), packed ``[T, H, D]`` rows ``[axes, T]``; int32 or int64. Pairs are ``(i, i + R / 2)``, or neighbours with ``interleaved``; columns
    from ``R`` on are copied. Tokens with a position outside the tables on any axis come out as zeros, which
    ``flash_sparse_attn.check_status()`` reports (status 5).

    Returns new tensors ``(query, key)``, or ``query`` alone with ``key=None``; gradients flow to both, not to the tables.
    Results are computed in fp32 and rounded once; no host synchronisation."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(apply_rotary_axes_func)(query, key, cos, sin, position_ids, sections, axes_dealt, interleaved, skip_checks)
    if not query.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    sections = tuple(sections)
    host = _lib.native() if _unseen() and isinstance(cos, torch.Tensor) and cos.ndim == 2 else None
    if host is not None:
        res = host.rotary_axes(query, key, cos, sin, position_ids, axis_bits(sections, cos.shape[1], bool(axes_dealt)), len(sections), bool(interleaved))
        if res is not None:
            return res
    if not skip_checks:
        _check(query, key, cos, sin, position_ids, sections)
    bits = axis_bits(sections, cos.shape[1], bool(axes_dealt))
    q_out, k_out = _turn(query, key, cos, sin, position_ids, bits, len(sections), bool(interleaved), False)
    return q_out if key is None else (q_out, k_out)
