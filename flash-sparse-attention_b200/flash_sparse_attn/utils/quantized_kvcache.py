"""A key-value cache whose rows (one token of one KV head) carry scales of their own, so that nothing has to be calibrated: rows are
quantised as they are appended, read back as 16-bit rows for a prompt's attention, and read as they are by
``flash_sparse_attn.flash_dense_attn_with_quantized_kvcache_func``. Wrappers of ``fsa_kv_append_quantized`` and ``fsa_kv_read_quantized``;
the reference, whose quantisation is per tensor, has no counterpart.

A cache is four tensors: codes of keys and of values and their scales, contiguous (``blocks`` = sequences) or paged (``blocks`` = pages):

=========  ====================================  ==========================================  ========================================
           codes                                 scales                                      value of a code
=========  ====================================  ==========================================  ========================================
int8       int8 ``[blocks, slots, Hkv, D]``      fp32 ``[blocks, slots, Hkv, 1]``            ``code * s``, ``s = max|row| / 127``
e4m3       float8_e4m3fn, the same               fp32, the same                              ``code * s``, ``s = max|row| / 448``
4 bits     uint8 ``[blocks, slots, Hkv, D/2]``,  bf16 ``[blocks, slots, Hkv, groups, 2]``:   ``z + (code - 8) * s`` with
           columns 2i and 2i + 1 a byte          ``(s, z)`` of each group of 32 or 64        ``s = (max - min) / 15``, ``z = min + 8 s``
=========  ====================================  ==========================================  ========================================

``empty_kv_quantized`` lays out one whose heads have their rows side by side, which is what the decode reads fastest; any strides do
whose rows are contiguous and start on 16-byte boundaries."""

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from flash_sparse_attn import _lib
from flash_sparse_attn.ops.triton.rotary import check_tables, split_offsets
from flash_sparse_attn.ops.triton.rotary_axes import axis_bits, check_positions, position_strides

_F16 = (torch.float16, torch.bfloat16)
_FORMATS = {torch.int8: _lib.QC_INT8, torch.float8_e4m3fn: _lib.QC_E4M3, torch.uint8: _lib.QC_INT4}
MAX_HEAD_DIM = 128


def empty_kv_quantized(blocks: int, slots: int, heads_kv: int, head_dim: int, dtype: torch.dtype = torch.int8, group_size: int = 64,
                       device="cuda") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(key_cache, value_cache, key_scales, value_scales)`` of ``blocks`` pages (or sequences) of ``slots`` positions, all zeros. ``dtype``:
    ``torch.int8``, ``torch.float8_e4m3fn``, or ``torch.uint8`` for 4 bits in groups of ``group_size`` columns. The tensors are views
    ``[blocks, slots, heads_kv, ..]`` of memory in which every head has its rows of a block side by side."""
    assert dtype in _FORMATS, "dtype must be int8, float8_e4m3fn, or uint8 for 4 bits"
    assert 0 < head_dim <= MAX_HEAD_DIM and head_dim % 16 == 0, f"head_dim must be a multiple of 16 up to {MAX_HEAD_DIM}"
    width, words, kind = head_dim, (1,), torch.float32
    if dtype == torch.uint8:
        assert group_size in (32, 64) and head_dim % group_size == 0, "4 bits take groups of 32 or 64 columns that divide head_dim"
        width, words, kind = head_dim // 2, (head_dim // group_size, 2), torch.bfloat16
    codes = [torch.zeros((blocks, heads_kv, slots, width), dtype=torch.uint8, device=device).view(dtype).transpose(1, 2) for _ in range(2)]
    scales = [torch.zeros((blocks, heads_kv, slots) + words, dtype=kind, device=device).transpose(1, 2) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def check_quantized_cache(key_cache, value_cache, key_scales, value_scales, page_table, batch):
    """The cache's contract, shared by what writes and what reads it."""
    device = key_cache.device
    for t in (value_cache, key_scales, value_scales, page_table):
        assert t is None or t.device == device, "All inputs must be on the same device"
    assert key_cache.ndim == 4 and key_cache.shape == value_cache.shape, "key and value codes must share one shape [blocks, slots, heads, ..]"
    assert key_cache.dtype in _FORMATS and value_cache.dtype == key_cache.dtype, "codes must be int8, float8_e4m3fn, or uint8 for 4 bits"
    int4 = key_cache.dtype == torch.uint8
    head_dim = key_cache.shape[3] * (2 if int4 else 1)
    assert 0 < head_dim <= MAX_HEAD_DIM and head_dim % 16 == 0, f"head_dim must be a multiple of 16 up to {MAX_HEAD_DIM}"
    assert key_cache.shape[0] > 0 and key_cache.shape[1] > 0 and key_cache.shape[2] > 0, "the cache must not be empty"
    assert max(key_cache.shape) < 2**31, "blocks and slots must be below 2^31"
    for t in (key_scales, value_scales):
        assert t.shape[:3] == key_cache.shape[:3], "scales must have the blocks, slots and heads of the codes"
        if int4:
            assert t.dtype == torch.bfloat16 and t.ndim == 5 and t.shape[4] == 2, "4-bit scales must be bfloat16 [blocks, slots, heads, groups, 2]"
            assert t.shape[3] in (head_dim // 32, head_dim // 64) and head_dim % t.shape[3] == 0 and head_dim // t.shape[3] in (32, 64), (
                "4 bits take groups of 32 or 64 columns that divide head_dim")
            assert t.stride(4) == 1 and (t.shape[3] == 1 or t.stride(3) == 2), "a row's scales must be contiguous"
            assert t.data_ptr() % 4 == 0 and all(n == 1 or s % 2 == 0 for n, s in zip(t.shape[:3], t.stride())), "pairs of scales must lie on 4-byte boundaries"
        else:
            assert t.dtype == torch.float32 and t.ndim == 4 and t.shape[3] == 1, "8-bit scales must be float32 [blocks, slots, heads, 1]"
    assert key_scales.shape == value_scales.shape, "key and value scales must share one shape"
    for t in (key_cache, value_cache):
        assert t.stride(3) == 1 or t.shape[3] == 1, "rows must be contiguous along head_dim"
        assert t.data_ptr() % 16 == 0 and all(n == 1 or s % 16 == 0 for n, s in zip(t.shape[:3], t.stride())), "rows of codes must lie on 16-byte boundaries"
    for t in (key_cache, value_cache, key_scales, value_scales, page_table):
        assert t is None or all(n == 1 or s > 0 for n, s in zip(t.shape, t.stride())), "caches and page_table must not be expanded"
    if page_table is None:
        assert key_cache.shape[0] == batch, "a contiguous cache must have one row per sequence"
    else:
        assert page_table.dtype == torch.int32 and page_table.ndim == 2 and page_table.shape[0] == batch, "page_table must be int32 [batch, max_pages]"
        assert page_table.shape[1] > 0 and (page_table.shape[1] == 1 or page_table.stride(1) == 1), "page_table must have pages and unit stride"


def fill_quantized_cache(c, key_cache, value_cache, key_scales, value_scales, page_table):
    """The library's view of a cache."""
    c.k, c.v, c.k_scales, c.v_scales = (t.data_ptr() for t in (key_cache, value_cache, key_scales, value_scales))
    c.format = _FORMATS[key_cache.dtype]
    int4 = c.format == _lib.QC_INT4
    per = 2 if int4 else 1  # scales of a 32-bit word
    c.k_stride_b, c.k_stride_s, c.k_stride_h = key_cache.stride()[:3]
    c.v_stride_b, c.v_stride_s, c.v_stride_h = value_cache.stride()[:3]
    c.ks_stride_b, c.ks_stride_s, c.ks_stride_h = (s // per for s in key_scales.stride()[:3])
    c.vs_stride_b, c.vs_stride_s, c.vs_stride_h = (s // per for s in value_scales.stride()[:3])
    # (the stride of a dimension of one is anything)
    for i, d in enumerate("bsh"):
        if key_cache.shape[i] == 1:
            for n in ("k", "v", "ks", "vs"):
                setattr(c, f"{n}_stride_{d}", 0)
    c.heads_kv, c.head_dim = key_cache.shape[2], key_cache.shape[3] * (2 if int4 else 1)
    c.group = c.head_dim // key_scales.shape[3] if int4 else 0
    if page_table is None:
        c.capacity = key_cache.shape[1]
    else:
        c.page_table, c.page_table_stride = page_table.data_ptr(), page_table.stride(0)
        c.num_pages, c.page_size = key_cache.shape[:2]
        c.max_pages = page_table.shape[1]


def rows_ok(t):
    """Rows of 16 bits on 16-byte boundaries."""
    if t.numel() == 0:
        return True
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(n == 1 or s % 8 == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _strides(t):
    """(batch, position, head) strides in elements; packed tensors have no batch stride, dimensions of one have none that counts."""
    s = [0 if n == 1 else st for n, st in zip(t.shape, t.stride())]
    return (0, s[0], s[1]) if t.ndim == 3 else tuple(s[:3])


def _check_append(query, key_new, value_new, key_cache, value_cache, key_scales, value_scales, seqused_k, cos, sin, page_table, free_pages,
                  free_count, cu_seqlens_new, seqlen_offsets, position_ids, sections, out):
    device, ndim = key_new.device, 3 if cu_seqlens_new is not None else 4
    for t in (query, value_new, key_cache, seqused_k, free_pages, free_count, cu_seqlens_new, out):
        assert t is None or t.device == device, "All inputs must be on the same device"
    assert key_new.ndim == ndim and key_new.shape == value_new.shape, (
        "key_new and value_new must be [batch, new_tokens, heads, head_dim], or packed [tokens, heads, head_dim] with cu_seqlens_new")
    assert key_new.dtype in _F16 and value_new.dtype == key_new.dtype, "new rows must be float16 or bfloat16, of one dtype"
    assert seqused_k.dtype == torch.int32 and seqused_k.ndim == 1 and seqused_k.is_contiguous() and seqused_k.numel() > 0, (
        "seqused_k must be a contiguous int32 tensor [batch]")
    batch = seqused_k.numel()
    check_quantized_cache(key_cache, value_cache, key_scales, value_scales, page_table, batch)
    heads_kv, head_dim = key_cache.shape[2], key_cache.shape[3] * (2 if key_cache.dtype == torch.uint8 else 1)
    assert key_new.shape[-2:] == (heads_kv, head_dim), "the cache must have the heads and head_dim of the new rows"
    if cu_seqlens_new is None:
        assert key_new.shape[0] == batch, "seqused_k must have one entry per sequence"
    else:
        assert cu_seqlens_new.dtype == torch.int32 and cu_seqlens_new.is_contiguous() and tuple(cu_seqlens_new.shape) == (batch + 1,), (
            "cu_seqlens_new must be a contiguous int32 tensor [batch + 1]")
    if query is not None:
        assert cos is not None, "queries are only turned: without cos and sin there is nothing to do with them"
        assert query.dtype == key_new.dtype and query.ndim == ndim, "query must have the dtype and form of key_new"
        assert query.shape[:-2] == key_new.shape[:-2] and query.shape[-1] == head_dim, "query and key_new must agree in their tokens and head_dim"
        assert query.shape[-2] > 0 and query.shape[-2] % heads_kv == 0, "num_heads_q must be divisible by num_heads_kv"
    for t in (query, key_new, value_new, out):
        assert t is None or rows_ok(t), "rows must be contiguous along head_dim and lie on 16-byte boundaries"
    assert (cos is None) == (sin is None), "cos and sin must be given together"
    if cos is None:
        assert seqlen_offsets is None and position_ids is None and sections is None, "positions belong to cos and sin"
    else:
        check_tables(cos, sin, head_dim, device)
        assert cos.shape[1] % 8 == 0, "rotary_dim must be a multiple of 16"
        assert cos.dtype != torch.float32 or (cos.data_ptr() % 16 == 0 and sin.data_ptr() % 16 == 0 and (cos.shape[0] == 1 or cos.stride(0) % 4 == 0)), (
            "rows of the tables must lie on 16-byte boundaries")
    assert (position_ids is None) == (sections is None), "position_ids and sections must be given together"
    if position_ids is not None:
        assert seqlen_offsets is None, "position_ids replace seqlen_offsets"
        check_positions(position_ids, sections, key_new.shape[:-2], device)
    assert (free_pages is None) == (free_count is None), "free_pages and free_count must be given together"
    if free_pages is not None:
        assert page_table is not None, "free_pages belong to paged caches"
        assert free_pages.dtype == torch.int32 and free_pages.is_contiguous(), "free_pages must be a contiguous int32 tensor"
        assert free_count.dtype == torch.int32 and free_count.numel() == 1, "free_count must be int32 [1]"
    if out is not None:
        assert query is not None and out.shape == query.shape and out.dtype == query.dtype, "out must have the shape and dtype of query"
        assert all(n == 1 or s > 0 for n, s in zip(out.shape, out.stride())), "out must not be expanded"


def append_kv_quantized(query: Optional[torch.Tensor], key_new: torch.Tensor, value_new: torch.Tensor, key_cache: torch.Tensor,
                        value_cache: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor, seqused_k: torch.Tensor,
                        cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, page_table: Optional[torch.Tensor] = None,
                        free_pages: Optional[torch.Tensor] = None, free_count: Optional[torch.Tensor] = None,
                        cu_seqlens_new: Optional[torch.Tensor] = None, seqlen_offsets: Optional[Union[int, torch.Tensor]] = None,
                        position_ids: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None, axes_dealt: bool = False,
                        interleaved: bool = False, advance: bool = True, out: Optional[torch.Tensor] = None,
                        skip_checks: bool = False) -> Optional[torch.Tensor]:
    """``append_kv_rotary`` into a cache whose rows carry their own scales: new keys ``[B, T, Hkv, D]`` (16 bits) are turned by their
    position, they and the new values are quantised row by row and stored at slots ``seqused_k[b] .. + T``; ``query [B, T, Hq, D]`` is turned
    alike and returned in its own dtype (None without a query). With int32 ``cu_seqlens_new [B + 1]`` the new rows are packed
    ``[tokens, heads, D]``. Without ``cos`` and ``sin`` keys are stored as they are.

    The position of a token is its slot plus ``seqlen_offsets`` (an int, or int32 ``[B]``) or, with ``sections``, given by ``position_ids
    [axes, B, T]`` (packed ``[axes, tokens]``) as in ``flash_sparse_attn.apply_rotary_axes_func``. ``rotary_dim`` a multiple of 16.

    Pages, ``free_pages``, ``free_count``, rows without room (status 3) or whose slot has no row in the tables (status 5) and ``advance`` are
    those of ``append_kv_rotary``; a token whose ``position_ids`` lie outside the tables is stored with a key of zeros (status 5). A row (with
    4 bits a group) that holds an infinity or a NaN reads back as NaN. No host synchronisation; no gradients."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(append_kv_quantized)(
            query, key_new, value_new, key_cache, value_cache, key_scales, value_scales, seqused_k, cos, sin, page_table, free_pages, free_count,
            cu_seqlens_new, seqlen_offsets, position_ids, sections, axes_dealt, interleaved, advance, out, skip_checks)
    if not key_new.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    sections = None if sections is None else tuple(sections)
    axes = sections is not None and isinstance(cos, torch.Tensor) and cos.ndim == 2
    host = _lib.native() if axes or sections is None else None  # (sections without tables are for the checks below to refuse)
    if host is not None:
        res = host.append_quantized(query, key_new, value_new, key_cache, value_cache, key_scales, value_scales, seqused_k, cos, sin, page_table,
                                    free_pages, free_count, cu_seqlens_new, seqlen_offsets, position_ids,
                                    axis_bits(sections, cos.shape[1], bool(axes_dealt)) if axes else None, len(sections) if axes else 0,
                                    bool(interleaved), bool(advance), out)
        if res is not None:
            if type(res) is int:
                _lib.check(res, "fsa_kv_append_quantized")
            return None if res is True else res
    if not skip_checks:
        _check_append(query, key_new, value_new, key_cache, value_cache, key_scales, value_scales, seqused_k, cos, sin, page_table,
                      free_pages, free_count, cu_seqlens_new, seqlen_offsets, position_ids, sections, out)
    device, batch = key_new.device, seqused_k.numel()
    bits = None if position_ids is None else axis_bits(sections, cos.shape[1], bool(axes_dealt))
    own_buffer = out is None
    if query is not None and own_buffer:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if key_new.numel() == 0:
        return out
    a = _lib.FsaKvAppendQuantArgs()
    fill_quantized_cache(a.cache, key_cache, value_cache, key_scales, value_scales, page_table)
    a.k_new, a.v_new, a.seqused_k = key_new.data_ptr(), value_new.data_ptr(), seqused_k.data_ptr()
    a.k_stride_b, a.k_stride_s, a.k_stride_h = _strides(key_new)
    a.v_stride_b, a.v_stride_s, a.v_stride_h = _strides(value_new)
    if query is not None:
        a.q, a.q_out, a.heads_q = query.data_ptr(), out.data_ptr(), query.shape[-2]
        a.q_stride_b, a.q_stride_s, a.q_stride_h = _strides(query)
        a.q_out_stride_b, a.q_out_stride_s, a.q_out_stride_h = _strides(out)
    if cos is not None:
        a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
        a.table_rows, a.rotary_dim, a.table_stride = cos.shape[0], 2 * cos.shape[1], 0 if cos.shape[0] == 1 else cos.stride(0)
        a.table_dtype = _lib.dtype_code(cos.dtype)
    a.offset, offsets = split_offsets(seqlen_offsets, batch, device)
    a.seqlen_offsets = _lib.ptr(offsets)
    if position_ids is not None:
        a.position_ids, a.position_ids_int64 = position_ids.data_ptr(), int(position_ids.dtype == torch.int64)
        a.position_stride_a, a.position_stride_b, a.position_stride_s = position_strides(position_ids)
        ctypes.memmove(a.axis_bits, bits, 32)
        a.axes = len(sections)
    a.free_pages, a.free_count, a.cu_seqlens_new = _lib.ptr(free_pages), _lib.ptr(free_count), _lib.ptr(cu_seqlens_new)
    a.status = _lib.status_word(device).data_ptr()
    a.batch = batch
    if cu_seqlens_new is not None:
        a.total = key_new.shape[0]
    else:
        a.new_tokens = key_new.shape[1]
    a.dtype = _lib.dtype_code(key_new.dtype)
    a.interleaved, a.advance = int(interleaved), int(advance)
    lib = _lib.load()
    ints = lib.fsa_kv_append_quantized_workspace_ints(ctypes.byref(a))
    place_ws = torch.empty(ints, dtype=torch.int32, device=device) if ints else None
    a.place_ws = _lib.ptr(place_ws)
    with torch.cuda.device(device):
        rc = lib.fsa_kv_append_quantized(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_kv_append_quantized")
    for t in (key_cache, value_cache, key_scales, value_scales):
        _lib.written(t)
    if advance:
        _lib.written(seqused_k)
    if free_pages is not None:
        _lib.written(page_table)
        _lib.written(free_count)
    if query is not None and not own_buffer:
        _lib.written(out)
    return out


def _check_read(key_cache, value_cache, key_scales, value_scales, seqused_k, page_table, cu_seqlens, max_seqlen, total, dtype, out):
    device = key_cache.device
    assert (cu_seqlens is None) == (total is None) and (cu_seqlens is None) != (max_seqlen is None), (
        "give max_seqlen for padded rows, or cu_seqlens and total for packed ones")
    assert dtype in _F16, "dtype must be float16 or bfloat16"
    if cu_seqlens is not None:
        assert cu_seqlens.dtype == torch.int32 and cu_seqlens.ndim == 1 and cu_seqlens.numel() >= 2 and cu_seqlens.is_contiguous(), (
            "cu_seqlens must be a contiguous int32 tensor [batch + 1]")
        batch = cu_seqlens.numel() - 1
    else:
        batch = page_table.shape[0] if page_table is not None else key_cache.shape[0]
    assert 0 <= (total if max_seqlen is None else max_seqlen) < 2**31, "max_seqlen and total must be sizes"
    check_quantized_cache(key_cache, value_cache, key_scales, value_scales, page_table, batch)
    for t in (seqused_k, cu_seqlens):
        assert t is None or t.device == device, "All inputs must be on the same device"
    assert seqused_k is None or (seqused_k.dtype == torch.int32 and tuple(seqused_k.shape) == (batch,) and seqused_k.is_contiguous()), (
        "seqused_k must be a contiguous int32 tensor [batch]")
    if out is not None:
        shape = _read_shape(key_cache, batch, max_seqlen, total)
        for t in out:
            assert t.device == device and tuple(t.shape) == shape and t.dtype == dtype and rows_ok(t), (
                f"out must be two tensors of shape {shape} and dtype {dtype} with rows on 16-byte boundaries")
            assert all(n == 1 or s > 0 for n, s in zip(t.shape, t.stride())), "out must not be expanded"


def _read_shape(key_cache, batch, max_seqlen, total):
    rows = (key_cache.shape[2], key_cache.shape[3] * (2 if key_cache.dtype == torch.uint8 else 1))
    return ((batch, max_seqlen) if total is None else (total,)) + rows


def read_kv_quantized(key_cache: torch.Tensor, value_cache: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
                      seqused_k: Optional[torch.Tensor] = None, page_table: Optional[torch.Tensor] = None,
                      cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None, total: Optional[int] = None,
                      dtype: torch.dtype = torch.bfloat16, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                      skip_checks: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(key, value)`` in 16 bits out of such a cache: the first ``seqused_k[b]`` (int32 ``[B]``; None: all) positions of every sequence
    as ``[B, max_seqlen, Hkv, D]``, zeros behind them, or with int32 ``cu_seqlens [B + 1]`` packed ``[total, Hkv, D]``; packed rows outside
    every sequence, or behind its last position, are zeros. This is what the forward operators take for a prompt whose first part
    is in the cache. Positions on a page outside the pool read as zeros and are reported (status 3). Values are computed in
    fp32 and rounded once; no host synchronisation; no gradients. ``out``: two tensors to write to."""
    if torch.compiler.is_compiling():  # a launch is not for the compiler to trace: its graph is cut here
        return torch.compiler.disable(read_kv_quantized)(key_cache, value_cache, key_scales, value_scales, seqused_k, page_table, cu_seqlens,
                                                         max_seqlen, total, dtype, out, skip_checks)
    if not key_cache.is_cuda:
        raise RuntimeError("flash_sparse_attn (B200 build) only runs on CUDA tensors; there is no CPU path")
    host = _lib.native() if out is None and dtype in _F16 else None
    if host is not None:
        res = host.read_quantized(key_cache, value_cache, key_scales, value_scales, seqused_k, page_table, cu_seqlens, max_seqlen, total,
                                  dtype == torch.bfloat16)
        if res is not None:
            if type(res) is int:
                _lib.check(res, "fsa_kv_read_quantized")
            return res
    if not skip_checks:
        _check_read(key_cache, value_cache, key_scales, value_scales, seqused_k, page_table, cu_seqlens, max_seqlen, total, dtype, out)
    device = key_cache.device
    batch = cu_seqlens.numel() - 1 if cu_seqlens is not None else (page_table if page_table is not None else key_cache).shape[0]
    shape = _read_shape(key_cache, batch, max_seqlen, total)
    own_buffer = out is None
    k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2)) if own_buffer else out
    if k.numel() == 0:
        return k, v
    a = _lib.FsaKvReadQuantArgs()
    fill_quantized_cache(a.cache, key_cache, value_cache, key_scales, value_scales, page_table)
    a.k_out, a.v_out = k.data_ptr(), v.data_ptr()
    a.k_out_stride_b, a.k_out_stride_s, a.k_out_stride_h = _strides(k)
    a.v_out_stride_b, a.v_out_stride_s, a.v_out_stride_h = _strides(v)
    a.seqused_k, a.cu_seqlens = _lib.ptr(seqused_k), _lib.ptr(cu_seqlens)
    a.status = _lib.status_word(device).data_ptr()
    a.batch, a.seqlen, a.total = batch, max_seqlen or 0, total or 0
    a.dtype = _lib.dtype_code(dtype)
    with torch.cuda.device(device):
        rc = _lib.load().fsa_kv_read_quantized(ctypes.byref(a), _lib.current_stream_ptr(device))
    _lib.check(rc, "fsa_kv_read_quantized")
    if not own_buffer:
        _lib.written(k)
        _lib.written(v)
    return k, v
