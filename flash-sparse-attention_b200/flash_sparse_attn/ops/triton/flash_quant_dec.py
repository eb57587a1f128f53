"""Host launcher of the decode over a cache whose rows carry their own scales: checks, workspace, one call into the library. Shapes
alone decide the launch (no device data is read on the host, nothing synchronises)."""

import ctypes
from typing import Optional

import torch

from flash_sparse_attn import _lib
from flash_sparse_attn.ops.triton import assert_inputs
from flash_sparse_attn.utils.quantized_kvcache import check_quantized_cache, fill_quantized_cache, rows_ok


def _check(query, key, value, key_scales, value_scales, softmax_scale, page_table, gather_kv_indices, seqused_k, out, lse):
    device = query.device
    assert query.ndim == 3 and query.shape[1] > 0, "query must be [batch, heads, head_dim]"
    assert query.dtype in (torch.float16, torch.bfloat16), "Input dtype must be float16 or bfloat16"
    batch = query.shape[0]
    check_quantized_cache(key, value, key_scales, value_scales, page_table, batch)
    heads_kv, head_dim = key.shape[2], key.shape[3] * (2 if key.dtype == torch.uint8 else 1)
    assert query.shape[1] % heads_kv == 0, "num_heads_q must be divisible by num_heads_kv"
    assert query.shape[2] == head_dim, "query and the cache must have one head_dim"
    assert rows_ok(query), "rows of query must be contiguous along head_dim and lie on 16-byte boundaries"
    if page_table is not None:
        assert_inputs._check_paged(key.shape[1], None, page_table, batch)
    assert_inputs._same_device(device, key, gather_kv_indices, seqused_k, out, lse)
    assert_inputs._int32(seqused_k, what="seqused_k")
    assert seqused_k is None or (tuple(seqused_k.shape) == (batch,) and seqused_k.is_contiguous()), "seqused_k must be [batch]"
    if gather_kv_indices is not None:
        assert_inputs._int32(gather_kv_indices, what="gather_kv_indices")
        assert gather_kv_indices.ndim == 2 and gather_kv_indices.shape[0] == batch, "gather_kv_indices must be [batch, topk]"
        assert gather_kv_indices.shape[1] <= 1 or gather_kv_indices.stride(1) == 1, "gather_kv_indices must have unit stride"
    assert softmax_scale is None or 0.0 < softmax_scale < float("inf"), "softmax_scale must be positive and finite"
    assert_inputs.check_out_buffers(out, lse, query.shape, query.dtype, query.shape[:2])
    for t in (out, lse):
        assert t is None or all(n == 1 or st > 0 for n, st in zip(t.shape, t.stride())), "out and lse must not be expanded"
    assert out is None or (out.data_ptr() % 4 == 0 and all(n == 1 or st % 2 == 0 for n, st in zip(out.shape[:2], out.stride()))), (
        "rows of out must lie on 4-byte boundaries")


def _strides(t):
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:2], t.stride()[:2]))


def attn_decode_quantized(query, key, value, key_scales, value_scales, softmax_scale: Optional[float] = None, page_table=None,
                          gather_kv_indices=None, seqused_k=None, out=None, lse=None, skip_checks=False):
    """Returns ``(out, lse)``."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(attn_decode_quantized)(query, key, value, key_scales, value_scales, softmax_scale, page_table,
                                                             gather_kv_indices, seqused_k, out, lse, skip_checks)
    if not query.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    host = _lib.native()
    if host is not None:
        res = host.decode_quantized(query, key, value, key_scales, value_scales, softmax_scale, page_table, gather_kv_indices, seqused_k, out, lse)
        if res is not None:
            if type(res) is int:
                _lib.check(res, "fsa_decode_quantized")
            return res
    if not skip_checks:
        _check(query, key, value, key_scales, value_scales, softmax_scale, page_table, gather_kv_indices, seqused_k, out, lse)
    device = query.device
    batch, heads_q, head_dim = query.shape
    given = out, lse
    if out is None:
        out = torch.empty((batch, heads_q, head_dim), dtype=query.dtype, device=device)
    if lse is None:
        lse = torch.empty((batch, heads_q), dtype=torch.float32, device=device)
    if batch == 0:
        return out, lse
    a = _lib.FsaQuantDecodeArgs()
    fill_quantized_cache(a.cache, key, value, key_scales, value_scales, page_table)
    a.q, a.out, a.lse = query.data_ptr(), out.data_ptr(), lse.data_ptr()
    a.q_stride_b, a.q_stride_h = _strides(query)
    a.o_stride_b, a.o_stride_h = _strides(out)
    a.lse_stride_b, a.lse_stride_h = _strides(lse)
    a.seqused_k = _lib.ptr(seqused_k)
    if gather_kv_indices is not None:
        # (an empty choice is not the absence of one; its address may be null)
        a.gather_kv_indices = gather_kv_indices.data_ptr() or out.data_ptr()
        a.topk, a.gather_stride = gather_kv_indices.shape[1], gather_kv_indices.stride(0)
    a.status = _lib.status_word(device).data_ptr()
    a.batch, a.heads_q, a.dtype = batch, heads_q, _lib.dtype_code(query.dtype)
    a.softmax_scale = float(softmax_scale) if softmax_scale is not None else head_dim**-0.5
    lib = _lib.load()
    with torch.cuda.device(device):
        nbytes = lib.fsa_decode_quantized_workspace_bytes(ctypes.byref(a))
        _lib.check(min(nbytes, 0), "fsa_decode_quantized")
        room = torch.empty(nbytes // 4, dtype=torch.float32, device=device)
        a.ws = room.data_ptr()
        rc = lib.fsa_decode_quantized(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_decode_quantized")
    for t in given:
        if t is not None:
            _lib.written(t)
    return out, lse
