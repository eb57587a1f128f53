"""Rotary positions with several axes against the definition in 64 bits: forms of pairs and of sections, odd sizes, strides, gradients,
positions outside the tables, other streams and captured calls; and refusals."""

import ctypes

import pytest
import torch

from test_rotary import check, done, launcher, normal, tables, turn  # noqa: F401

DEV = "cuda"


def owners(sections, dealt):
    """The axis of every pair, by dealing them out one at a time."""
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    for i in range(sum(sections)):
        a = i % len(sections)
        # an axis other than the first has its pairs at i = a, a + axes, ..; the first one takes the others too
        if a and left[a] == 0:
            a = 0
        left[a] -= 1
        out.append(a)
    assert left == [0] * len(sections)
    return out


def angles(table, ids, sections, dealt):
    """Rows of a table [.., R / 2] whose columns come from the positions of their axes; ids [axes, ..]."""
    own = owners(sections, dealt)
    return torch.stack([table.cpu()[ids[a].long().cpu(), i] for i, a in enumerate(own)], dim=-1)


def ids_for(seed, axes, rows, *lead, dtype=torch.int64):
    return torch.randint(0, rows, (axes,) + lead, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


FORMS = [(128, 128, (16, 24, 24), False), (128, 128, (24, 20, 20), True), (128, 64, (8, 8, 16), False), (96, 96, (16, 16, 16), False),
         (80, 80, (20, 20), True), (64, 20, (4, 3, 2, 1), False), (40, 24, (6, 3, 3), True), (24, 24, (5, 7), False), (16, 6, (1, 1, 1), True),
         (7, 4, (1, 1), False), (256, 256, (40, 40, 48), False)]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim,rotary_dim,sections,dealt", FORMS)
def test_forms_and_sizes(head_dim, rotary_dim, sections, dealt, dtype, interleaved):
    import flash_sparse_attn as fsa

    cos, sin = tables(61, rotary_dim // 2)
    ids = ids_for(6, len(sections), 61, 2, 33)
    q, k = normal(1, 2, 33, 6, head_dim, dtype=dtype).requires_grad_(), normal(2, 2, 33, 2, head_dim, dtype=dtype).requires_grad_()
    gq, gk = normal(3, *q.shape, dtype=dtype), normal(4, *k.shape, dtype=dtype)
    kw = dict(axes_dealt=dealt, interleaved=interleaved)
    oq, ok = fsa.apply_rotary_axes_func(q, k, cos, sin, ids, sections, **kw)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    done()
    c, s = angles(cos, ids, sections, dealt), angles(sin, ids, sections, dealt)
    for got, x, sign in ((oq, q, 1), (ok, k, 1), (dq, gq, -1), (dk, gk, -1)):
        check(got.detach(), *turn(x.detach(), c, s, interleaved, sign))
    # the gradient against a difference: the map is linear, so <g, f(x + e) - f(x)> = <g, f(e)> = <grad, e>
    e = normal(5, *q.shape, dtype=dtype)
    fe = fsa.apply_rotary_axes_func(e, None, cos, sin, ids, sections, **kw)
    left, right = (gq.double() * fe.double()).sum(), (dq.double() * e.double()).sum()
    # each side's elements are rounded once
    room = torch.finfo(dtype).eps * ((gq.double() * fe.double()).abs().sum() + (dq.double() * e.double()).abs().sum())
    assert (left - right).abs() <= room


@pytest.mark.gpu
def test_equal_positions_are_those_of_one_axis():
    import flash_sparse_attn as fsa

    cos, sin = tables(50, 32)
    q, k = normal(1, 2, 50, 4, 64), normal(2, 2, 50, 2, 64)
    one = torch.arange(50, device=DEV).expand(2, 50)
    want = fsa.apply_rotary_func(q, k, cos, sin)
    for sections, dealt in (((8, 12, 12), False), ((12, 10, 10), True)):
        got = fsa.apply_rotary_axes_func(q, k, cos, sin, one.expand(3, 2, 50), sections, axes_dealt=dealt)
        done()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["ids32", "shared", "packed", "strided ids", "strided heads", "one token"])
def test_forms_of_rows_and_positions(how, table):
    import flash_sparse_attn as fsa

    cos, sin = tables(31, 24, table)
    sections = (8, 8, 8)
    lead = {"packed": (57,), "one token": (1, 1)}.get(how, (3, 19))
    q, k = normal(1, *lead, 4, 48), normal(2, *lead, 2, 48)
    if how == "strided heads":
        both = normal(1, *lead, 9, 56)
        q, k = both[..., 1:5, 8:], both[..., 5:8:2, 8:]
    ids = ids_for(3, 3, 31, *lead, dtype=torch.int32 if how == "ids32" else torch.int64)
    if how == "shared":
        ids = ids[:, :1]
    if how == "strided ids":
        ids = ids_for(3, 3, 31, 19, 6).transpose(1, 2)[:, ::2]
    q.requires_grad_()
    oq, ok = fsa.apply_rotary_axes_func(q, k, cos, sin, ids, sections)
    oq.sum().backward()
    done()
    at = ids.expand(3, *lead)
    c, s = angles(cos, at, sections, False), angles(sin, at, sections, False)
    check(oq.detach(), *turn(q.detach(), c, s, False))
    check(ok, *turn(k, c, s, False))
    check(q.grad, *turn(torch.ones_like(q).detach(), c, s, False, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,rotary_dim,sections,dealt", [(128, 64, (8, 12, 12), False), (24, 24, (4, 4, 4), True), (7, 4, (1, 1), False)])
def test_many_tokens(head_dim, rotary_dim, sections, dealt):
    """Enough elements for threads that take several heads of a token each, and heads that do not come out even: 7 and 3."""
    import flash_sparse_attn as fsa

    total = 148 * 2048 // 30 + 53
    cos, sin = tables(997, rotary_dim // 2)
    ids = ids_for(4, len(sections), 997, 3, total)
    q, k = normal(1, 3, total, 7, head_dim).requires_grad_(), normal(2, 3, total, 3, head_dim)
    oq, ok = fsa.apply_rotary_axes_func(q, k, cos, sin, ids, sections, axes_dealt=dealt)
    g = normal(3, *q.shape)
    (dq,) = torch.autograd.grad(oq, q, g)
    done()
    c, s = angles(cos, ids, sections, dealt), angles(sin, ids, sections, dealt)
    for got, x, sign in ((oq, q, 1), (ok, k, 1), (dq, g, -1)):
        check(got.detach(), *turn(x.detach(), c, s, False, sign))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 31, 2**40])
def test_positions_outside_the_tables(bad):
    import flash_sparse_attn as fsa

    cos, sin = tables(31, 16)
    q, k = normal(1, 2, 9, 4, 40), normal(2, 2, 9, 2, 40)
    ids = ids_for(3, 3, 31, 2, 9)
    good = fsa.apply_rotary_axes_func(q, k, cos, sin, ids, (4, 6, 6))
    done()
    ids[2, 1, 4] = bad
    oq, ok = fsa.apply_rotary_axes_func(q, k, cos, sin, ids, (4, 6, 6))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status 5"):
        fsa.check_status()
    for got, want in zip((oq, ok), good):
        want[1, 4] = 0
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_gradients_of_one_tensor_and_of_gradients():
    import flash_sparse_attn as fsa

    cos, sin = tables(20, 16)
    ids = ids_for(3, 2, 20, 1, 20)
    q, k = normal(1, 1, 20, 2, 32).requires_grad_(), normal(2, 1, 20, 1, 32).requires_grad_()
    c, s = angles(cos, ids, (8, 8), False), angles(sin, ids, (8, 8), False)
    how = (cos, sin, ids, (8, 8))
    g = normal(3, 1, 20, 1, 32)
    (dk,) = torch.autograd.grad(fsa.apply_rotary_axes_func(q.detach(), k, *how)[1], k, g)
    check(dk, *turn(g, c, s, False, -1))
    (dk,) = torch.autograd.grad(fsa.apply_rotary_axes_func(q, k, *how)[1], k, g)
    check(dk, *turn(g, c, s, False, -1))
    gq = normal(4, 1, 20, 2, 32).requires_grad_()
    (dq,) = torch.autograd.grad(fsa.apply_rotary_axes_func(q, None, *how), q, gq, create_graph=True)
    h = normal(5, 1, 20, 2, 32)
    (dd,) = torch.autograd.grad(dq, gq, h)
    done()
    check(dd, *turn(h, c, s, False))
    # broadcast: one key row for the whole batch gets the sum of its gradients
    row = normal(6, 1, 20, 1, 32).requires_grad_()
    out = fsa.apply_rotary_axes_func(row.expand(3, 20, 1, 32), None, cos, sin, ids, (8, 8))
    out.backward(torch.ones_like(out))
    one = turn(torch.ones_like(row).detach(), c, s, False, -1)
    eps = torch.finfo(torch.bfloat16).eps
    # three equal 16-bit terms: each rounded once, added up in 16 bits with two more roundings
    assert ((row.grad.double().cpu() - 3 * one[0]).abs() <= 3 * eps * 3 * one[1] + 1e-6).all()


@pytest.mark.gpu
def test_another_stream_and_a_captured_training_step():
    import flash_sparse_attn as fsa

    cos, sin = tables(40, 32)
    ids = ids_for(3, 3, 40, 2, 40)
    q, k = normal(1, 2, 40, 4, 64).requires_grad_(), normal(2, 2, 40, 2, 64).requires_grad_()
    how, g = (cos, sin, ids, (8, 12, 12)), normal(3, 2, 40, 4, 64)
    side = torch.cuda.Stream()

    def step():  # (no eager graph of these leaves may live on another stream while a backward pass is captured: only values leave)
        oq, ok = fsa.apply_rotary_axes_func(q, k, *how)
        return (oq.detach(), ok.detach()) + torch.autograd.grad((oq, ok), (q, k), (g, torch.ones_like(ok)))

    want = step()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        q.mul_(2), k.mul_(2), ids.copy_(ids.flip(2))
    graph.replay()
    after = step()
    done()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(after, kept):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty_rows_and_inference_mode():
    import flash_sparse_attn as fsa

    cos, sin = tables(5, 16)
    q = torch.empty(2, 0, 4, 32, dtype=torch.bfloat16, device=DEV)
    assert fsa.apply_rotary_axes_func(q, None, cos, sin, torch.empty(2, 2, 0, dtype=torch.int64, device=DEV), (8, 8)).shape == q.shape
    with torch.inference_mode():
        x = normal(1, 1, 5, 2, 32)
        ids = ids_for(2, 2, 5, 1, 5)
        y = fsa.apply_rotary_axes_func(x, None, cos, sin, ids, (8, 8))
    done()
    check(y, *turn(x, angles(cos, ids, (8, 8), False), angles(sin, ids, (8, 8), False), False))


def test_sections_are_dealt_as_described():
    from flash_sparse_attn.ops.triton.rotary_axes import axis_bits

    for sections, dealt in (((16, 24, 24), False), ((24, 20, 20), True), ((1, 1), True), ((5, 2, 2, 3), True), ((128 - 3, 1, 1, 1), False)):
        word = int.from_bytes(axis_bits(sections, sum(sections), dealt), "little")
        assert [word >> 2 * i & 3 for i in range(sum(sections))] == owners(sections, dealt)


def test_refusals_on_the_cpu():
    import flash_sparse_attn as fsa
    from flash_sparse_attn import _lib
    from flash_sparse_attn.ops.triton import rotary_axes

    q, k, ids = torch.zeros(2, 5, 4, 32, dtype=torch.bfloat16), torch.zeros(2, 5, 2, 32, dtype=torch.bfloat16), torch.zeros(3, 2, 5, dtype=torch.int64)
    cos, sin = tables(9, 16, device="cpu")
    good = dict(query=q, key=k, cos=cos, sin=sin, position_ids=ids, sections=(4, 6, 6))
    rotary_axes._check(**good)
    rotary_axes._check(**dict(good, position_ids=ids[:, :1].int()))
    rotary_axes._check(**dict(good, query=q[0], key=k[0], position_ids=ids[:, 0]))
    for bad in (dict(query=q.float()), dict(query=q[0, 0]), dict(key=k[:, :4]), dict(key=k.half()), dict(key=k[..., :16]), dict(position_ids=ids[:2]),
                dict(position_ids=ids[:, :, :4]), dict(position_ids=ids[0]), dict(position_ids=ids.float()), dict(position_ids=None), dict(cos=cos[:, :8]),
                dict(query=torch.zeros(2, 5, 4, 264, dtype=torch.bfloat16), key=None), dict(cos=cos.double(), sin=sin.double()),
                dict(sections=(8, 8)), dict(query=q[0], key=k[0])):
        with pytest.raises(AssertionError):
            rotary_axes._check(**dict(good, **bad))
    for sections, pairs, dealt in (((16,), 16, False), ((4, 4, 4, 2, 2), 16, False), ((4, 6, 5), 16, False), ((0, 16), 16, False), ((-1, 17), 16, False),
                                   ((4, 12), 16, True), ((4.0, 12.0), 16, False), ((65, 64), 129, False)):
        with pytest.raises(AssertionError):
            rotary_axes.axis_bits(sections, pairs, dealt)
    with pytest.raises(RuntimeError, match="CUDA"):
        fsa.apply_rotary_axes_func(q, k, cos, sin, ids, (4, 6, 6))
    lib = _lib.load()

    def call(bits=0, **kw):
        a = _lib.FsaRotaryAxesArgs()
        a.q = a.q_out = a.cos = a.sin = a.status = a.position_ids = 256
        a.batch, a.seqlen, a.heads_q, a.head_dim, a.rotary_dim, a.table_rows, a.axes = 1, 1, 1, 64, 64, 1, 2
        a.dtype, a.table_dtype = _lib.DT_BF16, _lib.DT_F32
        a.axis_bits[1] = bits
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.fsa_rotary_axes(ctypes.byref(a), None)

    for kw in (dict(q=None), dict(status=None), dict(cos=None), dict(position_ids=None), dict(sin=258), dict(q=257), dict(rotary_dim=63),
               dict(rotary_dim=66), dict(rotary_dim=0), dict(table_rows=0), dict(batch=0), dict(heads_q=0), dict(heads_k=1), dict(seqlen=-1),
               dict(table_dtype=2), dict(axes=0), dict(axes=5), dict(bits=2), dict(bits=3 << 30)):
        assert call(**kw) == -1, kw
    assert call(dtype=_lib.DT_F32) == -2 and call(head_dim=272) == -2 and call(seqlen=0) == 0
    assert call(batch=1 << 20, seqlen=2047, heads_q=1 << 9) == -2


def test_argument_blocks_match_the_header():
    import os
    import re

    from flash_sparse_attn import _lib

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fsa_b200.h")).read()
    for name in ("FsaRotaryAxesArgs", "FsaQuantCache", "FsaKvAppendQuantArgs", "FsaKvReadQuantArgs", "FsaQuantDecodeArgs"):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1), flags=re.S)
        body = re.sub(r"\[\d+\]", "", body)
        fields = [re.findall(r"[A-Za-z_]\w*", part)[-1] for stmt in body.split(";") if stmt.strip() for part in stmt.split(",")]
        assert fields == [f[0] for f in getattr(_lib, name)._fields_], name
