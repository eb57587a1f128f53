"""Rotary positions, with their gradient: what the queries and keys of an attention layer go through in front of the
operators of ``interface.py``. One kernel of the library (``fsa_rotary``) for both tensors and both directions; the reference
leaves this step to its caller.

``append_kv_rotary`` of ``flash_sparse_attn.utils.kvcache`` applies the same rotation on the way into a KV cache."""

import ctypes
from typing import Optional, Tuple, Union

import torch

from flash_sparse_attn import _lib

_F16 = (torch.float16, torch.bfloat16)
_TABLE = (torch.float32, torch.float16, torch.bfloat16)


def check_tables(cos, sin, head_dim, device):
    """The tables' contract, shared with ``append_kv_rotary``."""
    assert isinstance(cos, torch.Tensor) and isinstance(sin, torch.Tensor), "cos and sin must be tensors [positions, rotary_dim / 2]"
    assert cos.ndim == 2 and cos.shape == sin.shape, "cos and sin must have one shape [positions, rotary_dim / 2]"
    assert cos.dtype == sin.dtype and cos.dtype in _TABLE, "cos and sin must be float32, float16 or bfloat16, of one dtype"
    assert cos.device == device and sin.device == device, "All inputs must be on the same device"
    assert cos.shape[0] > 0 and 0 < 2 * cos.shape[1] <= head_dim, "cos and sin must hold positions, and rotary_dim must not exceed head_dim"
    assert cos.stride() == sin.stride() and (cos.shape[1] == 1 or cos.stride(1) == 1), "cos and sin must share one layout with contiguous rows"
    assert not cos.requires_grad and not sin.requires_grad, "no gradient flows to cos and sin"


def split_offsets(seqlen_offsets, batch, device):
    """``seqlen_offsets`` as (int for all sequences, int32 tensor [batch] or None)."""
    if seqlen_offsets is None:
        return 0, None
    if isinstance(seqlen_offsets, torch.Tensor):
        assert seqlen_offsets.dtype == torch.int32 and tuple(seqlen_offsets.shape) == (batch,) and seqlen_offsets.is_contiguous(), (
            "seqlen_offsets must be an int or a contiguous int32 tensor [batch]")
        assert seqlen_offsets.device == device, "All inputs must be on the same device"
        return 0, seqlen_offsets
    offset = int(seqlen_offsets)
    assert -(2**31) <= offset < 2**31, "seqlen_offsets must fit 32 bits"
    return offset, None


def _check(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens):
    packed = cu_seqlens is not None
    assert query.ndim in ((3,) if packed else (3, 4)), "query must be [batch, seqlen, heads, head_dim] or packed [tokens, heads, head_dim]"
    assert packed or query.ndim == 4 or position_ids is not None, "packed tokens need cu_seqlens or position_ids"
    assert query.dtype in _F16, "Input dtype must be float16 or bfloat16"
    if key is not None:
        assert key.dtype == query.dtype, "All inputs must have the same dtype"
        assert key.ndim == query.ndim and key.shape[:-2] == query.shape[:-2] and key.shape[-1] == query.shape[-1], (
            "query and key must agree in their tokens and head_dim")
        assert key.device == query.device, "All inputs must be on the same device"
    check_tables(cos, sin, query.shape[-1], query.device)
    if packed:
        assert cu_seqlens.dtype == torch.int32 and cu_seqlens.ndim == 1 and cu_seqlens.numel() >= 2 and cu_seqlens.is_contiguous(), (
            "cu_seqlens must be a contiguous int32 tensor [batch + 1]")
        assert cu_seqlens.device == query.device, "All inputs must be on the same device"
    if position_ids is not None:
        assert not packed and seqlen_offsets is None, "position_ids replace cu_seqlens and seqlen_offsets"
        assert position_ids.dtype in (torch.int32, torch.int64), "position_ids must be int32 or int64"
        assert position_ids.device == query.device, "All inputs must be on the same device"
        tokens = tuple(query.shape[:-2])
        shared = (1, query.shape[1]) if query.ndim == 4 else tokens  # one row of positions for the whole batch
        assert tuple(position_ids.shape) in (tokens, shared), "position_ids must have one entry per token"


def _rows(t):
    """The tensor itself where its heads' columns lie side by side, else a copy that does."""
    return t if t is None or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(t):
    """(batch, position, head) strides in elements; packed tensors have no batch stride."""
    return (0, t.stride(0), t.stride(1)) if t.ndim == 3 else t.stride()[:3]


def _launch(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved, transposed):
    device = query.device
    query, key = _rows(query), _rows(key)
    q_out = torch.empty(query.shape, dtype=query.dtype, device=device)
    k_out = None if key is None else torch.empty(key.shape, dtype=key.dtype, device=device)
    a = _lib.FsaRotaryArgs()
    a.q, a.q_out, a.cos, a.sin = query.data_ptr(), q_out.data_ptr(), cos.data_ptr(), sin.data_ptr()
    a.k, a.k_out = _lib.ptr(key), _lib.ptr(k_out)
    a.status = _lib.status_word(device).data_ptr()
    a.q_stride_b, a.q_stride_s, a.q_stride_h = _strides(query)
    a.q_out_stride_b, a.q_out_stride_s, a.q_out_stride_h = _strides(q_out)
    if key is not None:
        a.k_stride_b, a.k_stride_s, a.k_stride_h = _strides(key)
        a.k_out_stride_b, a.k_out_stride_s, a.k_out_stride_h = _strides(k_out)
    if cu_seqlens is not None:
        a.batch, a.total, a.cu_seqlens = cu_seqlens.numel() - 1, query.shape[0], cu_seqlens.data_ptr()
    elif query.ndim == 4:
        a.batch, a.seqlen = query.shape[:2]
    else:
        a.batch, a.seqlen = 1, query.shape[0]
    a.offset, offsets = split_offsets(seqlen_offsets, a.batch, device)
    a.seqlen_offsets = _lib.ptr(offsets)
    if position_ids is not None:
        a.position_ids, a.position_ids_int64 = position_ids.data_ptr(), int(position_ids.dtype == torch.int64)
        if position_ids.ndim == 2:
            a.position_stride_b = 0 if position_ids.shape[0] == 1 else position_ids.stride(0)
        a.position_stride_s = position_ids.stride(-1)
    a.heads_q, a.head_dim = query.shape[-2:]
    a.heads_k = 0 if key is None else key.shape[-2]
    a.table_rows, a.rotary_dim, a.table_stride = cos.shape[0], 2 * cos.shape[1], cos.stride(0)
    a.dtype, a.table_dtype = _lib.dtype_code(query.dtype), _lib.dtype_code(cos.dtype)
    a.interleaved, a.transposed = int(interleaved), int(transposed)
    if q_out.numel() or (k_out is not None and k_out.numel()):
        with torch.cuda.device(device):
            rc = _lib.load().fsa_rotary(ctypes.byref(a), _lib.current_stream_ptr(device))
        _lib.check(rc, "fsa_rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The rotation with its gradient: the transposed rotation of the gradients, which is a rotation again and has a gradient too."""

    @staticmethod
    def forward(ctx, query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved, transposed):
        ctx.save_for_backward(cos, sin, position_ids, cu_seqlens, seqlen_offsets if isinstance(seqlen_offsets, torch.Tensor) else None)
        ctx.offset = None if isinstance(seqlen_offsets, torch.Tensor) else seqlen_offsets
        ctx.interleaved, ctx.transposed = interleaved, transposed
        ctx.set_materialize_grads(False)
        return _launch(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved, transposed)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, position_ids, cu_seqlens, offsets = ctx.saved_tensors
        dq, dk = (g if needed else None for g, needed in zip((dq, dk), ctx.needs_input_grad))
        how = (cos, sin, ctx.offset if offsets is None else offsets, position_ids, cu_seqlens, ctx.interleaved, not ctx.transposed)
        if dq is not None:
            dq, dk = _turn(dq, dk, *how)
        elif dk is not None:  # a launch's first tensor is the one that is there
            dk = _turn(dk, None, *how)[0]
        return (dq, dk) + (None,) * 7


def _turn(query, key, *how):
    if not _unseen() or (torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))):
        return _Rotary.apply(query, key, *how)
    return _launch(query, key, *how)


def _unseen() -> bool:
    """Whether no transform, dual number or trace wants to see what runs. Those see the Function, which has no tangents and says so."""
    return not (torch._C._are_functorch_transforms_active() or torch.autograd.forward_ad._current_level >= 0
                or torch._C._get_tracing_state() is not None)


def apply_rotary_func(
    query: torch.Tensor,
    key: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    seqlen_offsets: Optional[Union[int, torch.Tensor]] = None,
    position_ids: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    skip_checks: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Turn ``query [B, S, Hq, D]`` and ``key [B, S, Hkv, D]`` (16 bits, or packed ``[T, H, D]`` with int32 ``cu_seqlens
    [B + 1]``) by their positions. ``cos`` / ``sin [positions, R / 2]`` (fp32, or 16 bits) turn the first ``R`` columns of every
    head: pairs ``(i, i + R / 2)``, or neighbours ``(2i, 2i + 1)`` with ``interleaved``; the other columns are copied.

    A token's position is its place in its sequence plus ``seqlen_offsets`` (an int, or int32 ``[B]``), or its entry of
    ``position_ids`` (int32 / int64, ``[B, S]``, ``[1, S]`` or ``[T]``). Packed tokens outside every sequence come out as zeros,
    and so do tokens whose position is outside the tables, which ``flash_sparse_attn.check_status()`` reports (status 5).

    Returns new tensors ``(query, key)``, or ``query`` alone with ``key=None``; gradients flow to both, not to the tables.
    Results are computed in fp32 and rounded once; no host synchronisation."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(apply_rotary_func)(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved, skip_checks)
    if not query.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    host = _lib.native() if _unseen() else None
    if host is not None:
        res = host.rotary(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved)
        if res is not None:
            return res
    if not skip_checks:
        _check(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens)
    q_out, k_out = _turn(query, key, cos, sin, seqlen_offsets, position_ids, cu_seqlens, interleaved, False)
    return q_out if key is None else (q_out, k_out)
