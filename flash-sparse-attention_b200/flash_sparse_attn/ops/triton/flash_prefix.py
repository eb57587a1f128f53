"""Host launcher of the decode over a shared prefix: checks, workspaces, one call into the library. Shapes alone decide the launch (no device data is read on the host, nothing synchronises)."""

import ctypes
from typing import Optional

import torch

from flash_sparse_attn import _lib
from flash_sparse_attn.ops.triton import assert_inputs


def _rows_ok(t):
    """Rows that TMA can fetch: on 16-byte boundaries, none on top of another."""
    if t.numel() == 0:
        return True
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _check(query, key, value, prefix_key, prefix_value, softmax_scale, page_table, seqused_k, prefix_page_table, prefix_seqused, out, lse):
    device = query.device
    assert query.ndim == 3, "query must be [batch, heads, head_dim]"
    batch, heads_q, head_dim = query.shape
    assert key.ndim == 4 and key.shape == value.shape, "key and value must be [batch, seqlen, heads, head_dim], or pages with page_table"
    heads_kv = key.shape[2]
    assert_inputs._check_qkv(query, key, value, None, None, None, heads_q, heads_kv, head_dim, False, device)
    assert key.shape[3] == head_dim, "query, key and value must have one head_dim"
    if page_table is None:
        assert key.shape[0] == batch, "key and value must have one row per sequence"
    else:
        assert_inputs._check_paged(key.shape[1], None, page_table, batch)
        assert page_table.shape[1] > 0 and key.shape[0] > 0, "page_table and the pool must not be empty"
    assert prefix_key.shape == prefix_value.shape, "prefix_key and prefix_value must have one shape"
    assert prefix_key.dtype == prefix_value.dtype == query.dtype, "All inputs must have the same dtype"
    if prefix_page_table is None:
        assert prefix_key.ndim == 3, "prefix_key must be [seqlen, heads, head_dim], or pages with prefix_page_table"
    else:
        assert prefix_key.ndim == 4 and prefix_key.shape[0] > 0, "prefix_key must be pages [pages, page_size, heads, head_dim]"
        assert_inputs._check_paged(prefix_key.shape[1], None)
        assert prefix_page_table.ndim == 1 and prefix_page_table.is_contiguous(), "prefix_page_table must be a contiguous int32 tensor [max_pages]"
    assert prefix_key.shape[-2:] == key.shape[-2:], "the prefix must have the heads and head_dim of key"
    for t in (query, key, value, prefix_key, prefix_value):
        assert _rows_ok(t), "rows must be contiguous along head_dim, lie on 16-byte boundaries and not be expanded"
    assert_inputs._same_device(device, prefix_key, prefix_value, page_table, seqused_k, prefix_page_table, prefix_seqused, out, lse)
    assert_inputs._int32(page_table, prefix_page_table, what="page_table and prefix_page_table")
    assert_inputs._int32(seqused_k, prefix_seqused, what="seqused_k and prefix_seqused")
    assert seqused_k is None or (tuple(seqused_k.shape) == (batch,) and seqused_k.is_contiguous()), "seqused_k must be [batch]"
    assert prefix_seqused is None or prefix_seqused.numel() == 1, "prefix_seqused must have one element"
    assert softmax_scale is None or 0.0 < softmax_scale < float("inf"), "softmax_scale must be positive and finite"
    assert_inputs.check_out_buffers(out, lse, query.shape, query.dtype, query.shape[:2])
    for t in (out, lse):
        assert t is None or all(n == 1 or st > 0 for n, st in zip(t.shape, t.stride())), "out and lse must not be expanded"


def attn_decode_shared_prefix(query, key, value, prefix_key, prefix_value, softmax_scale: Optional[float] = None, page_table=None,
                              seqused_k=None, prefix_page_table=None, prefix_seqused=None, out=None, lse=None, skip_checks=False):
    """Returns ``(out, lse)``."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(attn_decode_shared_prefix)(query, key, value, prefix_key, prefix_value, softmax_scale, page_table, seqused_k,
                                                                 prefix_page_table, prefix_seqused, out, lse, skip_checks)
    if not query.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    host = _lib.native()
    if host is not None:
        res = host.shared_prefix(query, key, value, prefix_key, prefix_value, softmax_scale, page_table, seqused_k, prefix_page_table,
                                 prefix_seqused, out, lse)
        if res is not None:
            if type(res) is int:
                _lib.check(res, "fsa_decode_shared_prefix")
            return res
    if not skip_checks:
        _check(query, key, value, prefix_key, prefix_value, softmax_scale, page_table, seqused_k, prefix_page_table, prefix_seqused,
               out, lse)
    device = query.device
    batch, heads_q, head_dim = query.shape
    if out is None:
        out = torch.empty((batch, heads_q, head_dim), dtype=query.dtype, device=device)
    if lse is None:
        lse = torch.empty((batch, heads_q), dtype=torch.float32, device=device)
    if batch == 0:
        return out, lse
    a = _lib.FsaSharedPrefixArgs()
    a.q, a.k, a.v, a.prefix_k, a.prefix_v = (t.data_ptr() for t in (query, key, value, prefix_key, prefix_value))
    a.out, a.lse, a.status = out.data_ptr(), lse.data_ptr(), _lib.status_word(device).data_ptr()
    a.seqused_k, a.prefix_seqused = _lib.ptr(seqused_k), _lib.ptr(prefix_seqused)
    a.q_stride_b, a.q_stride_h = query.stride(0), query.stride(1)
    a.o_stride_b, a.o_stride_h = out.stride(0), out.stride(1)
    a.lse_stride_b, a.lse_stride_h = lse.stride(0), lse.stride(1)
    a.k_stride_b, a.k_stride_s, a.k_stride_h = key.stride()[:3]
    a.v_stride_b, a.v_stride_s, a.v_stride_h = value.stride()[:3]
    a.prefix_k_stride_s, a.prefix_k_stride_h = prefix_key.stride()[-3:-1]
    a.prefix_v_stride_s, a.prefix_v_stride_h = prefix_value.stride()[-3:-1]
    a.batch, a.heads_q, a.heads_kv, a.head_dim = batch, heads_q, key.shape[2], head_dim
    if page_table is None:
        a.seqlen_k = key.shape[1]
    else:
        page_table = page_table.contiguous()
        a.page_table, a.max_pages = page_table.data_ptr(), page_table.shape[1]
        a.num_pages, a.page_size = key.shape[:2]
    if prefix_page_table is None:
        a.prefix_seqlen = prefix_key.shape[0]
    elif prefix_page_table.numel():  # an empty table: a prefix of no keys
        a.prefix_page_table, a.prefix_max_pages = prefix_page_table.data_ptr(), prefix_page_table.numel()
        a.prefix_num_pages, a.prefix_page_size = prefix_key.shape[:2]
        a.prefix_k_stride_p, a.prefix_v_stride_p = prefix_key.stride(0), prefix_value.stride(0)
    a.dtype = _lib.dtype_code(query.dtype)
    a.softmax_scale = float(softmax_scale) if softmax_scale is not None else head_dim**-0.5
    lib = _lib.load()
    ws = _lib.FsaSharedPrefixWorkspace()
    with torch.cuda.device(device):
        _lib.check(lib.fsa_shared_prefix_workspace_bytes(ctypes.byref(a), ctypes.byref(ws)), "fsa_shared_prefix_workspace_bytes")
        room = torch.empty((ws.out_partial + ws.sum_partial + ws.plan_ws) // 4, dtype=torch.float32, device=device)
        a.out_partial = room.data_ptr()
        a.sum_partial = a.out_partial + ws.out_partial
        a.plan_ws = a.sum_partial + ws.sum_partial
        rc = lib.fsa_decode_shared_prefix(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_decode_shared_prefix")
    return out, lse
