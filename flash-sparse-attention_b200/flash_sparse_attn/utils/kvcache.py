"""Device-side steps in front of a (top-k) decode: appending the new key / value rows to the cache, with the rotary
positions on the way or without, and cutting global top-k positions down to one shard of a sharded cache. Thin wrappers of ``fsa_kv_append``,
``fsa_kv_append_rotary`` and ``fsa_localize_indices``; none has a counterpart in the reference, which leaves cache management to its caller
(the cache layouts are the ones its decode operators read: contiguous ``[B, Sk, Hkv, D]`` or paged
``[pages, page_size, Hkv, D]`` with ``page_table [B, max_pages]``)."""

import ctypes
from typing import Optional, Union

import torch

from flash_sparse_attn import _lib
from flash_sparse_attn.ops.triton.rotary import check_tables, split_offsets
from flash_sparse_attn.utils.quantized_kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized  # noqa: F401


def append_kv(key_new: torch.Tensor, value_new: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
              seqused_k: torch.Tensor, page_table: Optional[torch.Tensor] = None,
              free_pages: Optional[torch.Tensor] = None, free_count: Optional[torch.Tensor] = None,
              pos_ws: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Write ``key_new / value_new [B, T, Hkv, D]`` at positions ``seqused_k[b] .. + T`` of the cache and advance
    ``seqused_k`` (int32 [B], in place). Paged caches take missing pages (page-table entries < 0) from the stack
    ``free_pages`` (int32) of height ``free_count`` (int32 [1], decremented in place). Rows without room are dropped
    and reported by ``flash_sparse_attn.check_status()`` (status 3). No host synchronisation. Returns ``seqused_k``."""
    if not key_new.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    device = key_new.device
    batch, new_tokens, heads_kv, head_dim = key_new.shape
    assert value_new.shape == key_new.shape and value_new.stride() == key_new.stride()
    assert value_cache.shape == key_cache.shape and value_cache.stride() == key_cache.stride()
    assert key_cache.dtype == key_new.dtype == value_new.dtype == value_cache.dtype
    assert seqused_k.dtype == torch.int32 and seqused_k.numel() == batch and seqused_k.is_contiguous()
    assert key_new.stride(-1) == 1 and key_cache.stride(-1) == 1
    if pos_ws is None:
        pos_ws = torch.empty(batch, dtype=torch.int32, device=device)
    a = _lib.FsaKvAppendArgs()
    a.k_new, a.v_new, a.k_cache, a.v_cache = (t.data_ptr() for t in (key_new, value_new, key_cache, value_cache))
    a.seqused_k, a.pos_ws = seqused_k.data_ptr(), pos_ws.data_ptr()
    a.page_table, a.free_pages, a.free_count = _lib.ptr(page_table), _lib.ptr(free_pages), _lib.ptr(free_count)
    a.status = _lib.status_word(device).data_ptr()
    a.new_stride_b, a.new_stride_s, a.new_stride_h = key_new.stride(0), key_new.stride(1), key_new.stride(2)
    a.cache_stride_b, a.cache_stride_s, a.cache_stride_h = key_cache.stride(0), key_cache.stride(1), key_cache.stride(2)
    a.batch, a.new_tokens, a.heads_kv, a.head_dim = batch, new_tokens, heads_kv, head_dim
    if page_table is not None:
        assert page_table.dtype == torch.int32 and page_table.shape[0] == batch and page_table.stride(1) == 1
        a.page_size, a.page_table_stride = key_cache.shape[1], page_table.stride(0)
    else:
        a.capacity = key_cache.shape[1]
    a.dtype = _lib.dtype_code(key_new.dtype)
    with torch.cuda.device(device):
        rc = _lib.load().fsa_kv_append(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_kv_append")
    _lib.written(seqused_k)
    return seqused_k


_F16 = (torch.float16, torch.bfloat16)
_FP8 = (torch.float8_e4m3fn, torch.float8_e5m2)


def _check_append(query, key_new, value_new, key_cache, value_cache, seqused_k, cos, sin, page_table, free_pages, free_count,
                  cu_seqlens_new, query_scale, key_scale, value_scale, out):
    device, ndim = key_new.device, 3 if cu_seqlens_new is not None else 4
    for t in (query, value_new, key_cache, value_cache, seqused_k, page_table, free_pages, free_count, cu_seqlens_new, out):
        assert t is None or t.device == device, "All inputs must be on the same device"
    assert key_new.ndim == ndim and key_new.shape == value_new.shape, (
        "key_new and value_new must be [batch, new_tokens, heads, head_dim], or packed [tokens, heads, head_dim] with cu_seqlens_new")
    for t in (key_cache, value_cache, seqused_k, page_table, free_pages, out):
        assert t is None or all(n == 1 or s > 0 for n, s in zip(t.shape, t.stride())), "what is written, and page_table, must not be expanded"
    heads_kv, head_dim = key_new.shape[-2:]
    assert key_new.dtype in _F16 and value_new.dtype == key_new.dtype, "new rows must be float16 or bfloat16, of one dtype"
    if query is not None:
        assert query.dtype == key_new.dtype and query.ndim == ndim, "query must have the dtype and form of key_new"
        assert query.shape[:-2] == key_new.shape[:-2] and query.shape[-1] == head_dim, "query and key_new must agree in their tokens and head_dim"
        assert query.shape[-2] % heads_kv == 0, "num_heads_q must be divisible by num_heads_kv"
    for t in (query, key_new, value_new, key_cache, value_cache):
        assert t is None or t.shape[-1] == 1 or t.stride(-1) == 1, "rows must be contiguous along head_dim"
    assert key_cache.ndim == 4 and key_cache.shape == value_cache.shape and key_cache.dtype == value_cache.dtype, (
        "key_cache and value_cache must share one shape and dtype")
    assert key_cache.shape[2:] == key_new.shape[-2:], "the cache must have the heads and head_dim of the new rows"
    scales = (query_scale if query is not None else key_scale, key_scale, value_scale)
    if key_cache.dtype in _FP8:
        for t in scales:
            assert isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.numel() == 1 and t.device == device, (
                "an FP8 cache needs query_scale, key_scale and value_scale, fp32 tensors of one element")
    else:
        assert key_cache.dtype == key_new.dtype, "the cache must be of the new rows' dtype, or FP8"
        assert query_scale is None and key_scale is None and value_scale is None, "scales belong to FP8 caches"
    assert seqused_k.dtype == torch.int32 and seqused_k.ndim == 1 and seqused_k.is_contiguous(), "seqused_k must be a contiguous int32 tensor [batch]"
    batch = seqused_k.numel()
    if cu_seqlens_new is None:
        assert key_new.shape[0] == batch, "seqused_k must have one entry per sequence"
    else:
        assert cu_seqlens_new.dtype == torch.int32 and cu_seqlens_new.is_contiguous() and tuple(cu_seqlens_new.shape) == (batch + 1,), (
            "cu_seqlens_new must be a contiguous int32 tensor [batch + 1]")
    if page_table is None:
        assert key_cache.shape[0] == batch, "a contiguous cache must have one row per sequence"
        assert free_pages is None and free_count is None, "free_pages belong to paged caches"
    else:
        assert page_table.dtype == torch.int32 and page_table.ndim == 2 and page_table.shape[0] == batch, "page_table must be int32 [batch, max_pages]"
        assert page_table.shape[1] == 1 or page_table.stride(1) == 1, "page_table must have unit stride"
        assert page_table.shape[1] > 0 and key_cache.shape[0] > 0 and key_cache.shape[1] > 0, "the cache must have pages"
        assert (free_pages is None) == (free_count is None), "free_pages and free_count must be given together"
        if free_pages is not None:
            assert free_pages.dtype == torch.int32 and free_pages.is_contiguous(), "free_pages must be a contiguous int32 tensor"
            assert free_count.dtype == torch.int32 and free_count.numel() == 1, "free_count must be int32 [1]"
    check_tables(cos, sin, head_dim, device)
    if out is not None:
        assert query is not None and out.shape == query.shape and (out.shape[-1] == 1 or out.stride(-1) == 1), "out must have the shape of query"
        assert out.dtype == (key_cache.dtype if key_cache.dtype in _FP8 else query.dtype), "out must have the dtype of the rotated query"


def append_kv_rotary(query: Optional[torch.Tensor], key_new: torch.Tensor, value_new: torch.Tensor, key_cache: torch.Tensor,
                     value_cache: torch.Tensor, seqused_k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                     page_table: Optional[torch.Tensor] = None, free_pages: Optional[torch.Tensor] = None,
                     free_count: Optional[torch.Tensor] = None, cu_seqlens_new: Optional[torch.Tensor] = None,
                     seqlen_offsets: Optional[Union[int, torch.Tensor]] = None, interleaved: bool = False,
                     query_scale: Optional[torch.Tensor] = None, key_scale: Optional[torch.Tensor] = None,
                     value_scale: Optional[torch.Tensor] = None, advance: bool = True, out: Optional[torch.Tensor] = None,
                     skip_checks: bool = False) -> Optional[torch.Tensor]:
    """``append_kv`` with the rotary positions applied on the way: new keys ``[B, T, Hkv, D]`` are turned by their position and
    stored with the new values at slots ``seqused_k[b] .. + T`` of the cache, ``query [B, T, Hq, D]`` is turned alike and returned
    (None without a query). With int32 ``cu_seqlens_new [B + 1]`` the new rows are packed ``[tokens, heads, D]``. ``cos`` / ``sin``
    and ``interleaved`` are those of ``flash_sparse_attn.apply_rotary_func``; the position of a token is its slot plus
    ``seqlen_offsets`` (an int, or int32 ``[B]``: the length of a prefix that lies elsewhere).

    A cache in FP8 takes 16-bit rows divided by ``key_scale`` / ``value_scale`` (fp32, one element), rounded and saturated; the
    query then comes back in the cache's dtype, divided by ``query_scale``: what the ``*_with_kvcache_func`` operators take with
    ``is_quant=True``.

    Missing pages (page-table entries < 0) come off the top of the stack ``free_pages`` (int32) of height ``free_count`` (int32
    [1], in place), in the order of sequences and slots. Rows without room (status 3) or without a row in the tables (status 5) are
    not stored, nor are the rows behind them in their sequence, and their query rows come out as zeros;
    ``flash_sparse_attn.check_status()`` reports it, and until it has been asked forward, backward and shared-prefix calls write no results. ``seqused_k`` (int32 [B]) grows by the rows stored, in place; with
    ``advance=False`` it stays, for layers that share the lengths: all but the last. No host synchronisation; no gradients."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(append_kv_rotary)(
            query, key_new, value_new, key_cache, value_cache, seqused_k, cos, sin, page_table, free_pages, free_count, cu_seqlens_new,
            seqlen_offsets, interleaved, query_scale, key_scale, value_scale, advance, out, skip_checks)
    if not key_new.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    host = _lib.native()
    if host is not None:
        res = host.append(query, key_new, value_new, key_cache, value_cache, seqused_k, cos, sin, page_table, free_pages, free_count,
                          cu_seqlens_new, seqlen_offsets, interleaved, query_scale, key_scale, value_scale, advance, out)
        if res is not None:
            if type(res) is int:
                _lib.check(res, "fsa_kv_append_rotary")
            return None if res is True else res
    if not skip_checks:
        _check_append(query, key_new, value_new, key_cache, value_cache, seqused_k, cos, sin, page_table, free_pages, free_count,
                      cu_seqlens_new, query_scale, key_scale, value_scale, out)
    device, fp8 = key_new.device, key_cache.dtype in _FP8
    batch = seqused_k.numel()
    own_buffer = out is None
    if query is not None and own_buffer:
        out = torch.empty(query.shape, dtype=key_cache.dtype if fp8 else query.dtype, device=device)
    if key_new.numel() == 0:
        return out
    a = _lib.FsaKvAppendRotaryArgs()

    def place(name, t):
        setattr(a, name + "_stride_b", 0 if t.ndim == 3 else t.stride(0))
        setattr(a, name + "_stride_s", t.stride(-3))
        setattr(a, name + "_stride_h", t.stride(-2))

    if query is not None:
        a.q, a.q_out, a.heads_q = query.data_ptr(), out.data_ptr(), query.shape[-2]
        place("q", query)
        place("q_out", out)
    a.k_new, a.v_new, a.k_cache, a.v_cache = (t.data_ptr() for t in (key_new, value_new, key_cache, value_cache))
    place("k", key_new)
    place("v", value_new)
    place("k_cache", key_cache)
    place("v_cache", value_cache)
    a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
    a.table_rows, a.rotary_dim, a.table_stride = cos.shape[0], 2 * cos.shape[1], cos.stride(0)
    a.seqused_k, a.cu_seqlens_new = seqused_k.data_ptr(), _lib.ptr(cu_seqlens_new)
    a.page_table, a.free_pages, a.free_count = _lib.ptr(page_table), _lib.ptr(free_pages), _lib.ptr(free_count)
    a.offset, offsets = split_offsets(seqlen_offsets, batch, device)
    a.seqlen_offsets = _lib.ptr(offsets)
    if fp8:
        a.q_scale, a.k_scale, a.v_scale = _lib.ptr(query_scale), key_scale.data_ptr(), value_scale.data_ptr()
    a.status = _lib.status_word(device).data_ptr()
    a.batch, a.heads_kv, a.head_dim = batch, key_new.shape[-2], key_new.shape[-1]
    if cu_seqlens_new is not None:
        a.total = key_new.shape[0]
    else:
        a.new_tokens = key_new.shape[1]
    if page_table is not None:
        a.num_pages, a.page_size = key_cache.shape[:2]
        a.max_pages, a.page_table_stride = page_table.shape[1], page_table.stride(0)
    else:
        a.capacity = key_cache.shape[1]
    a.dtype, a.cache_dtype, a.table_dtype = (_lib.dtype_code(t.dtype) for t in (key_new, key_cache, cos))
    a.interleaved, a.advance = int(interleaved), int(advance)
    ints = _lib.load().fsa_kv_append_rotary_workspace_ints(ctypes.byref(a))
    place_ws = torch.empty(ints, dtype=torch.int32, device=device) if ints else None
    a.place_ws = _lib.ptr(place_ws)
    with torch.cuda.device(device):
        rc = _lib.load().fsa_kv_append_rotary(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_kv_append_rotary")
    if advance:
        _lib.written(seqused_k)
    if not own_buffer:
        _lib.written(out)
    return out


def localize_indices(gather_kv_indices: torch.Tensor, key_bounds: torch.Tensor, out: Optional[torch.Tensor] = None,
                     count: Optional[torch.Tensor] = None):
    """Global top-k positions ``[B, topk]`` (int32) -> ``(local, count)``: per row the positions inside
    ``[lo, hi) = key_bounds[b]`` shifted by ``-lo``, moved to the front in their original order, the rest ``-1``;
    ``count [B]`` says how many. ``out`` / ``count`` may be supplied so that the call allocates nothing."""
    device = gather_kv_indices.device
    rows, topk = gather_kv_indices.shape
    assert gather_kv_indices.dtype == torch.int32 and gather_kv_indices.stride(1) == 1
    assert key_bounds.dtype == torch.int32 and tuple(key_bounds.shape) == (rows, 2) and key_bounds.is_contiguous()
    out = torch.empty((rows, topk), dtype=torch.int32, device=device) if out is None else out
    count = torch.empty(rows, dtype=torch.int32, device=device) if count is None else count
    with torch.cuda.device(device):
        rc = _lib.load().fsa_localize_indices(gather_kv_indices.data_ptr(), gather_kv_indices.stride(0),
                                              key_bounds.data_ptr(), out.data_ptr(), out.stride(0), count.data_ptr(),
                                              rows, topk, _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_localize_indices")
    return out, count
