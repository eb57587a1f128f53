"""Rotary positions against the definition in 64 bits: forms of pairs, odd sizes, strides, all ways to say where a token
stands, gradients, and refusals."""

import ctypes

import pytest
import torch

DEV = "cuda"


@pytest.fixture(params=["native", "python"], autouse=True)
def launcher(request, monkeypatch):
    """Every test runs through the native launcher and through the Python one."""
    from flash_sparse_attn import _lib

    _lib.load()
    if request.param == "python":
        monkeypatch.setattr(_lib, "_host", None)
    else:
        assert _lib.native() is not None


def tables(rows, half, dtype=torch.float32, device=DEV):
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device)


def turn(x, cos, sin, interleaved, sign=1.0):
    """x [.., H, D] and the tables' rows of its tokens [.., R / 2], in 64 bits; also the size of what was added up."""
    x, c, s = x.double().cpu(), cos.double().cpu()[..., None, :], sign * sin.double().cpu()[..., None, :]
    half = c.shape[-1]
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one], size[..., two] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def check(got, want, size):
    """One rounding to 16 bits (half a step, relative; half of the smallest step below the normal values) of an fp32 result
    whose two products and sum are off by at most 2^-24 each of what is added: 2^-22 covers the three."""
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * want.abs() * (1 + 2.0**-10) + 2.0**-22 * size + info.smallest_normal * info.eps / 2
    wrong = (got.double().cpu() - want).abs() > bound
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()} elements"


def normal(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def done():
    import flash_sparse_attn as fsa

    torch.cuda.synchronize()
    fsa.check_status()


SHAPES = [(128, 128), (128, 64), (64, 32), (96, 48), (80, 20), (40, 10), (24, 24), (16, 2), (7, 4), (112, 112), (256, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim,rotary_dim", SHAPES)
def test_forms_and_sizes(head_dim, rotary_dim, dtype, interleaved):
    import flash_sparse_attn as fsa

    cos, sin = tables(61, rotary_dim // 2)
    q, k = normal(1, 2, 33, 6, head_dim, dtype=dtype), normal(2, 2, 33, 2, head_dim, dtype=dtype)
    q.requires_grad_(), k.requires_grad_()
    gq, gk = normal(3, *q.shape, dtype=dtype), normal(4, *k.shape, dtype=dtype)
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin, seqlen_offsets=28, interleaved=interleaved)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    done()
    at = torch.arange(33) + 28
    for got, x, sign in ((oq, q, 1), (ok, k, 1), (dq, gq, -1), (dk, gk, -1)):
        check(got.detach(), *turn(x.detach(), cos[at], sin[at], interleaved, sign))
    # the gradient against a difference: the map is linear, so <g, f(x + e) - f(x)> = <g, f(e)> = <grad, e>
    e = normal(5, *q.shape, dtype=dtype)
    fe = fsa.apply_rotary_func(e, None, cos, sin, seqlen_offsets=28, interleaved=interleaved)
    left, right = (gq.double() * fe.double()).sum(), (dq.double() * e.double()).sum()
    # each side's elements are rounded once
    room = torch.finfo(dtype).eps * ((gq.double() * fe.double()).abs().sum() + (dq.double() * e.double()).abs().sum())
    assert (left - right).abs() <= room


@pytest.mark.gpu
@pytest.mark.parametrize("batch,seq,heads_q,heads_k", [(1, 1, 1, 1), (3, 1, 5, 1), (1, 4001, 20, 4), (70, 150, 32, 8)])
def test_lengths_from_one_token_on(batch, seq, heads_q, heads_k):
    import flash_sparse_attn as fsa

    cos, sin = tables(seq, 32)
    q, k = normal(1, batch, seq, heads_q, 64), normal(2, batch, seq, heads_k, 64)
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin)
    done()
    check(oq, *turn(q, cos[:seq], sin[:seq], False))
    check(ok, *turn(k, cos[:seq], sin[:seq], False))


@pytest.mark.gpu
@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["offsets", "ids64", "ids32", "shared ids", "packed", "packed offsets", "packed ids"])
def test_where_a_token_stands(how, table):
    import flash_sparse_attn as fsa

    b, s, rows = 4, 19, 131
    cos, sin = tables(rows, 24, table)
    g = torch.Generator().manual_seed(7)
    off = torch.randint(0, rows - s, (b,), generator=g).to(torch.int32)
    ids = torch.randint(0, rows, (b, s), generator=g)
    lens = [0, 5, 19, 0, 1, 13, 0]
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    if how.startswith("packed"):
        total = int(cu[-1]) + 6  # rows behind the last sequence
        q, k = normal(1, total, 4, 48), normal(2, total, 2, 48)
        at = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(6, dtype=torch.long)])
        if how == "packed ids":
            at = torch.randint(0, rows, (total,), generator=g)
            kw = dict(position_ids=at.to(DEV))
        else:
            kw = dict(cu_seqlens=cu.to(DEV))
            if how == "packed offsets":
                more = torch.randint(0, rows - 19, (len(lens),), generator=g).to(torch.int32)
                at = at + torch.cat([more.long().repeat_interleave(torch.tensor(lens)), torch.zeros(6, dtype=torch.long)])
                kw["seqlen_offsets"] = more.to(DEV)
    else:
        q, k = normal(1, b, s, 4, 48), normal(2, b, s, 2, 48)
        if how == "offsets":
            at, kw = torch.arange(s) + off[:, None], dict(seqlen_offsets=off.to(DEV))
        elif how == "shared ids":
            at, kw = ids[0].expand(b, s), dict(position_ids=ids[:1].to(DEV))
        else:
            at, kw = ids, dict(position_ids=ids.to(torch.int64 if how == "ids64" else torch.int32).to(DEV))
    q.requires_grad_()
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin, **kw)
    (dq,) = torch.autograd.grad(oq, q, q.detach())
    done()
    (yq, zq), (yk, zk), (yd, zd) = (turn(x.detach(), cos.cpu()[at], sin.cpu()[at], False, sg) for x, sg in ((q, 1), (k, 1), (q, -1)))
    if how in ("packed", "packed offsets"):
        for y in (yq, yk, yd):
            y[-6:] = 0
    check(oq.detach(), yq, zq)
    check(ok, yk, zk)
    check(dq, yd, zd)


@pytest.mark.gpu
def test_strided_inputs_and_gradients():
    import flash_sparse_attn as fsa

    b, s, hq, hk, d = 3, 37, 4, 2, 64
    cos, sin = tables(s, d // 2)
    fused = normal(1, b, s, (hq + 2 * hk) * d + 3)  # rows that start on odd elements
    q = fused[..., :hq * d].unflatten(-1, (hq, d))
    k = fused[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin)
    heads_first = normal(2, b, hq, s, d).transpose(1, 2)
    columns_last = normal(3, b, s, d, hk).transpose(2, 3)
    o2, o3 = fsa.apply_rotary_func(heads_first, columns_last, cos, sin)
    wide = tables(s, 40)
    cut = (wide[0][:, 3:3 + 32], wide[1][:, 3:3 + 32])  # table rows that are no multiple of 16 bytes apart and begin inside one
    o4 = fsa.apply_rotary_func(q, None, *cut)
    leaf = q.detach().clone().requires_grad_()
    out = fsa.apply_rotary_func(leaf, None, cos, sin)
    # broadcast gradients (stride 0), and gradients in another layout
    (d1,) = torch.autograd.grad(out, leaf, torch.ones((), dtype=out.dtype, device=DEV).expand_as(out), retain_graph=True)
    (d2,) = torch.autograd.grad(out, leaf, heads_first)
    done()
    for got, x, (c, t), sign in ((oq, q, (cos, sin), 1), (ok, k, (cos, sin), 1), (o2, heads_first, (cos, sin), 1),
                                 (o3, columns_last, (cos, sin), 1), (o4, q, cut, 1), (d1, torch.ones_like(leaf), (cos, sin), -1),
                                 (d2, heads_first, (cos, sin), -1)):
        check(got, *turn(x.detach(), c, t, False, sign))


@pytest.mark.gpu
def test_only_what_is_asked_for():
    import flash_sparse_attn as fsa

    cos, sin = tables(9, 16)
    q, k = normal(1, 1, 9, 2, 32), normal(2, 1, 9, 1, 32).requires_grad_()
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin)
    (dk,) = torch.autograd.grad(ok, k, torch.ones_like(ok))
    done()
    check(dk, *turn(torch.ones_like(ok), cos, sin, False, -1))
    with torch.no_grad():
        assert not fsa.apply_rotary_func(k, None, cos, sin).requires_grad
    empty = fsa.apply_rotary_func(q[:, :0], None, cos, sin)
    assert empty.shape == (1, 0, 2, 32)
    # special values stay in their own pair
    x = torch.ones(1, 1, 1, 32, dtype=torch.bfloat16, device=DEV)
    x[..., 3], x[..., 5] = float("inf"), float("nan")
    y = fsa.apply_rotary_func(x, None, cos, sin, seqlen_offsets=2)
    assert torch.isfinite(y).sum() == 28 and torch.isnan(y[..., [5, 21]]).all() and torch.isinf(y[..., [3, 19]]).all()


@pytest.mark.gpu
def test_gradients_of_gradients():
    import flash_sparse_attn as fsa

    cos, sin = tables(9, 16)
    q, k, g = normal(1, 1, 9, 2, 32).requires_grad_(), normal(2, 1, 9, 1, 32).requires_grad_(), normal(3, 1, 9, 2, 32).requires_grad_()
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin)
    (dq,) = torch.autograd.grad(oq, q, g, create_graph=True)
    assert torch.autograd.grad(ok, q, torch.ones_like(ok), allow_unused=True, retain_graph=True) == (None,)
    h = normal(4, *q.shape)
    (dg,) = torch.autograd.grad(dq, g, h)
    done()
    check(dq.detach(), *turn(g.detach(), cos, sin, False, -1))
    check(dg, *turn(h, cos, sin, False))


@pytest.mark.gpu
def test_tangents_are_refused():
    """Forward mode has no rule here: it has to be told so, not to lose its tangents. Also in a gradient of gradients."""
    import torch.autograd.forward_ad as fw

    import flash_sparse_attn as fsa

    cos, sin = tables(9, 16)
    x, y = normal(1, 1, 9, 2, 32), normal(2, 1, 9, 2, 32).requires_grad_()
    out = fsa.apply_rotary_func(y, None, cos, sin)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for q, k in ((dual, None), (x, dual)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                fsa.apply_rotary_func(q, k, cos, sin)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.autograd.grad(out, y, dual)


@pytest.mark.gpu
def test_positions_outside_the_tables_are_reported():
    import flash_sparse_attn as fsa

    cos, sin = tables(10, 16)
    x = normal(1, 1, 12, 2, 32)
    y = fsa.apply_rotary_func(x, None, cos, sin, seqlen_offsets=-1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="device status 5"):
        fsa.check_status()
    assert not y[0, 0].any() and not y[0, 11:].any()
    check(y[:, 1:11], *turn(x[:, 1:11], cos, sin, False))


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    import flash_sparse_attn as fsa

    cos, sin = tables(50, 64)
    q, k = normal(1, 2, 50, 4, 128).requires_grad_(), normal(2, 2, 50, 2, 128).requires_grad_()
    gq, gk = normal(3, *q.shape), normal(4, *k.shape)

    def step():
        oq, ok = fsa.apply_rotary_func(q, k, cos, sin)
        return (oq.detach(), ok.detach(), *torch.autograd.grad((oq, ok), (q, k), (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        q.mul_(2), gk.mul_(4)  # exact in 16 bits
    graph.replay()
    done()
    for a, b, f in zip(got, want, (2, 1, 1, 4)):
        assert torch.equal(a, b * f)


def test_refusals():
    from flash_sparse_attn import _lib
    from flash_sparse_attn.ops.triton import rotary

    cos, sin = tables(10, 16, device="cpu")
    q, k = torch.zeros(2, 10, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 10, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)

    def ok(query=q, key=k, c=cos, s=sin, off=None, ids=None, cu_seqlens=None):
        rotary._check(query, key, c, s, off, ids, cu_seqlens)

    ok(), ok(ids=torch.zeros(2, 10, dtype=torch.int64)), ok(q[0], k[0], cu_seqlens=cu), ok(q[0], None, ids=torch.zeros(10, dtype=torch.int32))
    for bad in (dict(query=q.float()), dict(key=k.half()), dict(key=k[:, :9]), dict(key=k[..., :32]), dict(c=cos[:, :8]),
                dict(c=cos.double(), s=sin.double()), dict(query=q[..., :16], key=k[..., :16]), dict(query=q[0], key=k[0]),
                dict(cu_seqlens=cu), dict(query=q[0], key=k[0], cu_seqlens=cu.long()), dict(ids=torch.zeros(2, 9, dtype=torch.int64)),
                dict(ids=torch.zeros(2, 10)), dict(ids=torch.zeros(2, 10, dtype=torch.int32), off=1),
                dict(query=q[0], key=k[0], ids=torch.zeros(1, dtype=torch.int32)), dict(c=cos.T, s=sin.T),
                dict(c=cos.clone().requires_grad_()), dict(c=cos[:0], s=sin[:0]), dict(c=cos[:, :0], s=sin[:, :0])):
        with pytest.raises(AssertionError):
            ok(**bad)
    with pytest.raises(AssertionError):
        rotary.split_offsets(torch.zeros(3, dtype=torch.int32), 2, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary.apply_rotary_func(q, k, cos, sin)
    # the library's own checks, in front of any launch
    lib = _lib.load()

    def call(**kw):
        a = _lib.FsaRotaryArgs()
        a.q = a.q_out = a.cos = a.sin = a.status = 256
        a.batch, a.seqlen, a.heads_q, a.head_dim, a.rotary_dim, a.table_rows = 1, 1, 1, 64, 64, 1
        a.dtype, a.table_dtype = _lib.DT_BF16, _lib.DT_F32
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.fsa_rotary(ctypes.byref(a), None)

    for kw in (dict(q=None), dict(status=None), dict(cos=None), dict(sin=258), dict(q=257), dict(rotary_dim=63), dict(rotary_dim=66),
               dict(rotary_dim=0), dict(table_rows=0), dict(batch=0), dict(heads_q=0), dict(heads_k=1), dict(seqlen=-1), dict(table_dtype=2)):
        assert call(**kw) == -1, kw
    assert call(dtype=_lib.DT_F32) == -2 and call(seqlen=0) == 0 and call(batch=1 << 20, seqlen=2047, heads_q=1 << 9) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 5, "tensor"])
def test_packed_tokens_outside_every_sequence(offset):
    """Bounds that begin behind the first token and end in front of the last: those tokens are in no sequence and have no position,
    whatever is added to it. They come out as zeros, and so do their gradients."""
    import flash_sparse_attn as fsa

    cos, sin = tables(12, 16)
    q, k = normal(1, 11, 4, 32).requires_grad_(), normal(2, 11, 2, 32)
    cu = torch.tensor([3, 3, 5, 5, 9], dtype=torch.int32, device=DEV)
    more = [5, 3, 1, 7] if offset == "tensor" else [offset] * 4
    kw = dict(seqlen_offsets=torch.tensor(more, dtype=torch.int32, device=DEV) if offset == "tensor" else offset)
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin, cu_seqlens=cu, **kw)
    (dq,) = torch.autograd.grad(oq, q, torch.ones_like(oq))
    done()
    at = torch.tensor([more[1], more[1] + 1, *range(more[3], more[3] + 4)])
    for got, x, sign in ((oq.detach(), q.detach(), 1), (ok, k, 1), (dq, torch.ones_like(q), -1)):
        assert not got[:3].any() and not got[9:].any()
        check(got[3:9], *turn(x[3:9], cos[at], sin[at], False, sign))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim,rotary_dim,threads", [(128, 64, 8), (24, 24, 3), (40, 20, 10), (7, 4, 4)])
def test_many_tokens(head_dim, rotary_dim, threads, dtype, packed, interleaved):
    """Enough elements for threads that take several heads of a token each, and heads that do not come out even: 7 and 3."""
    import flash_sparse_attn as fsa

    total = 148 * 2048 // (10 * threads) + 53
    lens = [0, total // 3, 1, 0, total // 2, 17]
    lens.append(total - sum(lens) - 9)  # and nine tokens behind the last sequence
    if packed:
        lead, kw = (total,), dict(cu_seqlens=torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV))
        at = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(9, dtype=torch.long)]) + 2
    else:
        lead, kw, at = (2, (total + 1) // 2), {}, torch.arange((total + 1) // 2) + 2
    cos, sin = tables(int(at.max()) + 1, rotary_dim // 2)
    q, k = normal(1, *lead, 7, head_dim, dtype=dtype).requires_grad_(), normal(2, *lead, 3, head_dim, dtype=dtype).requires_grad_()
    gq, gk = normal(3, *q.shape, dtype=dtype), normal(4, *k.shape, dtype=dtype)
    oq, ok = fsa.apply_rotary_func(q, k, cos, sin, seqlen_offsets=2, interleaved=interleaved, **kw)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    done()
    for got, x, sign in ((oq, q, 1), (ok, k, 1), (dq, gq, -1), (dk, gk, -1)):
        want, size = turn(x.detach(), cos.cpu()[at], sin.cpu()[at], interleaved, sign)
        if packed:
            want[-9:] = 0
        check(got.detach(), want, size)
