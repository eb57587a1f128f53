"""A cache whose rows carry their own scales: what is stored, code for code, against the definition in single fp32 steps and against the
values in 64 bits; where it is stored; reading back; special values; other streams and captured calls; and refusals."""

import ctypes

import pytest
import torch

from test_append_rotary import pages_for
from test_rotary import check as check_turned
from test_rotary import done, launcher, normal, tables, turn  # noqa: F401
from test_rotary_axes import angles, ids_for

DEV = "cuda"
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "int4": torch.uint8}


def rotated(x, c, s, interleaved):
    """x [.., H, D] turned in fp32, every product and sum rounded by itself."""
    x, c, s = x.float().cpu(), c.float().cpu()[..., None, :], s.float().cpu()[..., None, :]
    half, y = c.shape[-1], x.clone()
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    return y


def quantised(x, kind, group=64):
    """Rows [.., D] in fp32 -> (codes, scales) as kept, step by step as defined."""
    if kind == "int4":
        g = x.unflatten(-1, (-1, group))
        low, high = g.amin(-1), g.amax(-1)
        s = ((high - low) / 15).to(torch.bfloat16)
        s = torch.where(s.float() < 2.0**-126, 0, s)
        z = (low + 8 * s.float()).to(torch.bfloat16)
        inverse = torch.where(s > 0, 1 / s.float(), 0)
        n = (((g - z.float()[..., None]) * inverse[..., None]).round().clamp(-8, 7) + 8).to(torch.uint8).flatten(-2)
        return n[..., 0::2] | n[..., 1::2] << 4, torch.stack([s, z], -1)
    top = 127.0 if kind == "int8" else 448.0
    s = x.abs().amax(-1, keepdim=True) / top
    s = torch.where(s < 2.0**-126, 0, s)
    n = (x * torch.where(s > 0, 1 / s, 0)).clamp(-top, top)
    return (n.round() if kind == "int8" else n).to(KINDS[kind]), s


def values(codes, scales):
    """What is kept stands for, in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    if codes.dtype != torch.uint8:
        return codes.float().double() * scales.double()
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8
    n = n.unflatten(-1, (scales.shape[-2], -1))
    return (n * scales[..., :1].double() + scales[..., 1:].double()).flatten(-2)


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def make_cache(seed, blocks, slots, hkv, d, kind, group=64, by_head=True):
    """Codes and scales with something in every place."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        shape = (blocks, hkv, slots, d) if by_head else (blocks, slots, hkv, d)
        c, s = quantised(torch.randn(shape, generator=g), kind, group)
        c, s = c.to(DEV), s.to(DEV)
        out.append((c.transpose(1, 2), s.transpose(1, 2)) if by_head else (c, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def run(new, used, kind, d=64, hq=4, hkv=2, dtype=torch.bfloat16, group=64, by_head=True, packed=False, page=0, slots=0, capacity=600, half=None,
        interleaved=False, offset=0, rows=700, stack=True, height=None, break_table=None, bad_page=None, sections=None, table_dtype=torch.float32,
        advance=True, behind=0, seed=0, spread=1.0):
    """One append, compared place by place with a plain one."""
    from flash_sparse_attn.utils.kvcache import append_kv_quantized

    b, total = len(new), sum(new) + behind
    q, k, v = (normal(i, total, h, d, dtype=dtype) * spread for i, h in ((1, hq), (2, hkv), (3, hkv)))
    table = free = None
    count = 0
    if page:
        pool, table, free, count = pages_for(torch.Generator().manual_seed(seed), used, slots, page)
        count = count if height is None else height
        if break_table is not None:
            table[break_table] = pool if bad_page is None else bad_page
        if not stack:
            free = None
        blocks, size = pool, page
    else:
        blocks, size = b, capacity
    cache = make_cache(seed, blocks, size, hkv, d, kind, group, by_head)
    want = [t.cpu().clone() for t in cache]
    half = d // 2 if half is None else half
    cos = sin = ids = None
    if half:
        cos, sin = tables(rows, half, table_dtype)
        if sections:
            ids = ids_for(9, len(sections), rows, total)
    # ---- the plain append
    left, pages, lengths, kept_rows = count, None if table is None else table.clone(), list(used), []
    oq = torch.zeros(total, hq, d, dtype=torch.float64)
    size_q, row = torch.zeros_like(oq), 0
    for i, n in enumerate(new):
        cap = size if table is None else slots * page
        reach = max(0, min(n, cap - used[i], rows - used[i] - offset if half and not sections else n))
        if used[i] < 0 or (half and not sections and used[i] + offset < 0):
            reach = 0
        kept = reach
        if table is not None and reach:
            for j in range(used[i] // page, (used[i] + reach - 1) // page + 1):
                if pages[i, j] < 0 and free is not None and left > 0:
                    left -= 1
                    pages[i, j] = free[left]
                if not 0 <= pages[i, j] < pool:
                    kept = min(kept, max(0, j * page - used[i]))
        kept_rows.append(kept)
        at = slice(row, row + kept)
        kk, vv = k[at].float().cpu(), v[at].float().cpu()
        if half:
            if sections:
                c, s = (angles(t, ids[:, at], sections, False) for t in (cos, sin))
            else:
                c, s = (t.cpu()[used[i] + offset:used[i] + offset + kept] for t in (cos, sin))
            kk = rotated(k[at], c, s, interleaved)
            oq[at], size_q[at] = turn(q[at], c, s, interleaved)
        for x, codes, scales in ((kk, want[0], want[2]), (vv, want[1], want[3])):
            n8, s8 = quantised(x, kind, group)
            for t in range(kept):
                slot = used[i] + t
                place = (i, slot) if table is None else (int(pages[i, slot // page]), slot % page)
                codes.view(torch.uint8)[place] = n8[t].view(torch.uint8)
                scales[place] = s8[t]
        if advance:
            lengths[i] += kept
        row += n
    # ---- the call
    used_d = torch.tensor(used, dtype=torch.int32, device=DEV)
    table_d = None if table is None else table.to(DEV)
    kw = dict(page_table=table_d, interleaved=interleaved, advance=advance)
    if free is not None:
        kw.update(free_pages=free.to(DEV), free_count=torch.tensor([count], dtype=torch.int32, device=DEV))
    if half and not sections:
        kw["seqlen_offsets"] = offset
    args = [q, k, v]
    if packed:
        kw["cu_seqlens_new"] = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    else:
        args = [x.view(b, new[0], *x.shape[1:]) for x in args]
    if sections:
        kw.update(position_ids=ids if packed else ids.view(len(sections), b, new[0]), sections=sections)
    if not half:
        args[0] = None
    got = append_kv_quantized(*args, *cache, used_d, cos, sin, **kw)
    torch.cuda.synchronize()
    for name, a, w in zip(("key codes", "value codes", "key scales", "value scales"), cache, want):
        assert torch.equal(bits(a), bits(w)), name
    assert used_d.tolist() == lengths
    if table is not None:
        assert table_d.tolist() == pages.tolist()
        if free is not None:
            assert kw["free_count"].item() == left
    if half:
        check_turned(got.reshape(oq.shape), oq, size_q)
    else:
        assert got is None
    return sum(new) - sum(kept_rows)


FORMS = [("int8", 128, 64), ("int8", 48, 64), ("int8", 16, 64), ("e4m3", 64, 64), ("e4m3", 112, 64), ("int4", 128, 64), ("int4", 128, 32), ("int4", 64, 64),
         ("int4", 96, 32), ("int4", 32, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,d,group", FORMS)
def test_codes_and_scales(kind, d, group, dtype):
    kw = dict(kind=kind, d=d, group=group, dtype=dtype)
    run([1, 1, 1], [0, 5, 599], **kw)
    run([3, 3], [0, 130], by_head=False, interleaved=True, offset=7, **kw)
    run([70, 0, 1, 33], [500, 3, 9, 0], packed=True, behind=3, half=8, **kw)
    run([50, 50], [0, 50], half=0, **kw)  # not turned
    done()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
def test_pages_and_axes(kind, group):
    import flash_sparse_attn as fsa

    kw = dict(kind=kind, d=128, group=group)
    # without a stack: the sequence of 32 rows has no page for the next one
    assert run([1] * 5, [0, 31, 32, 33, 127], page=32, slots=6, stack=False, break_table=(0, 0), bad_page=3, **kw) == 1
    with pytest.raises(RuntimeError, match="status 3"):
        fsa.check_status()
    run([1] * 5, [0, 31, 32, 33, 127], page=32, slots=6, **kw)
    run([100, 0, 1, 64], [0, 31, 32, 5], page=64, slots=4, packed=True, sections=(16, 24, 24), **kw)
    run([4, 4], [62, 64], page=64, slots=4, sections=(24, 20, 20), interleaved=True, **kw)
    run([4, 4], [62, 64], page=64, slots=4, table_dtype=torch.bfloat16, advance=False, by_head=False, **kw)
    done()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
@pytest.mark.parametrize("packed", [False, True])
def test_many_rows(kind, group, packed):
    """Enough elements for threads that take several heads of a row each, of 6 query, 2 key and 2 value heads."""
    new = [1300, 0, 1, 1700, 900] if packed else [1500, 1500, 1500]
    used = [5, 9, 63, 64, 0][:len(new)]
    run(new, used, kind, d=128, group=group, hq=6, hkv=2, packed=packed, page=64, slots=28, rows=1800, half=32, interleaved=packed, spread=3.0)
    done()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_rows_without_room_or_angles(kind):
    """A sequence keeps the rows in front of the first that has no place; the status word says why."""
    import flash_sparse_attn as fsa

    for why, lost, kw in ((3, 5, dict(new=[4, 4], used=[597, 598], capacity=600)), (3, 38, dict(new=[40, 2], used=[30, 0], page=32, slots=2, height=0, packed=True)),
                          (3, 1, dict(new=[1, 1], used=[64, 3], page=32, slots=2)), (5, 3, dict(new=[4, 1], used=[20, 3], rows=21, packed=True)),
                          (3, 1, dict(new=[1], used=[3], page=32, slots=2, break_table=(0, 0), stack=False)), (3, 2, dict(new=[2], used=[-1], half=0))):
        got = run(kind=kind, **kw)
        with pytest.raises(RuntimeError, match=f"status {why}"):
            fsa.check_status()
        assert got >= 1, (why, lost, kw)


@pytest.mark.gpu
def test_positions_outside_the_tables_give_keys_of_zeros():
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized

    cos, sin = tables(9, 32)
    q, k = normal(1, 2, 2, 4, 64), normal(2, 2, 2, 2, 64)
    ids = torch.zeros(2, 2, 2, dtype=torch.int32, device=DEV)
    ids[1, 0, 1] = 9
    for kind in KINDS.values():
        cache = empty_kv_quantized(2, 10, 2, 64, kind)
        used = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
        oq = append_kv_quantized(q, k, k, *cache, used, cos, sin, position_ids=ids, sections=(16, 16))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status 5"):
            fsa.check_status()
        assert used.tolist() == [5, 6] and not oq[0, 1].any() and oq[0, 0].any()
        assert not values(cache[0][0, 4], cache[2][0, 4]).any() and values(cache[1][0, 4], cache[3][0, 4]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
def test_special_rows(kind, group, dtype):
    """Zeros, constants, one outlier, the type's largest and smallest values, infinities and NaN: the row (the group) stands for what
    went in, to the format's own step, or for NaN."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    info, d = torch.finfo(dtype), 128
    x = normal(1, 12, d, dtype=dtype)
    x[0] = 0
    x[1] = 1.5
    x[2] = -3.0
    x[3, 77] = 1000.0
    x[4] *= float(torch.tensor(info.max / 8).to(dtype))
    x[5] = x[5].sign() * info.smallest_normal
    x[6, 5] = float("inf")
    x[7, 100] = float("nan")
    x[8, 0] = -float("inf")
    x[9] = x[9].abs() + 100
    cache = empty_kv_quantized(1, 12, 1, d, KINDS[kind], group_size=group)
    used = torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = x.view(1, 12, 1, d)
    append_kv_quantized(None, rows, rows.flip(-1).contiguous(), *cache, used)
    k, v = read_kv_quantized(*cache, used, max_seqlen=12, dtype=dtype)
    done()
    per = group if kind == "int4" else d
    for got, want in ((k[0, :, 0], x), (v[0, :, 0], x.flip(-1))):
        w = want.double().cpu().unflatten(-1, (-1, per))
        g = got.double().cpu().unflatten(-1, (-1, per))
        finite = w.isfinite().all(-1, keepdim=True)
        assert torch.equal(g.isnan(), (~finite).expand_as(g)), kind
        w, g = torch.where(finite, w, 0), torch.where(finite, g, 0)
        out = torch.finfo(dtype).eps / 2  # the result's own rounding
        tiny = 2.0**-126 * 448  # rows below are kept as zeros
        if kind == "int4":
            # half a step, and what rounding z and s to bf16 (2^-9) takes from the ends of the range, 15 steps wide
            step, mid = (w.amax(-1, keepdim=True) - w.amin(-1, keepdim=True)) / 15, w.abs().amax(-1, keepdim=True)
            bound = step * (0.5 + 15 * 2.0**-8) * 1.01 + 2.0**-8 * mid * 1.01
        elif kind == "int8":
            bound = w.abs().amax(-1, keepdim=True) / 127 * 0.501
        else:  # half of a step, relative; below the normal values 2^-6 / 448 of the largest half of 2^-9
            bound = torch.maximum(w.abs() * 2.0**-4, w.abs().amax(-1, keepdim=True) / 448 * 2.0**-10) * 1.001
        assert ((g - w).abs() <= bound + out * w.abs() * 1.1 + tiny + info.smallest_normal * info.eps).all(), kind
    fsa.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "e4m3", "int4"])
def test_rows_from_end_to_end_of_bf16(kind):
    """The largest and the least number of a row: their difference is beyond fp32, neither is an infinity."""
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    cache = empty_kv_quantized(1, 4, 1, 64, KINDS[kind])
    used = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = (torch.linspace(-3e38, 3e38, 64, device=DEV, dtype=torch.float64).to(torch.bfloat16)).view(1, 1, 1, 64)
    append_kv_quantized(None, x, x, *cache, used)
    got, _ = read_kv_quantized(*cache, used, max_seqlen=1)
    done()
    # half a step (of 15 over 6e38, of 254, or e4m3's 2^-4 of the value), and 2^-8 of 3e38 for each of the roundings of s (eight times), z and the result
    step = {"int4": 2e37 + 10 * 2.0**-8 * 3e38, "int8": 1.2e36 + 2.0**-8 * 3e38, "e4m3": 2.0**-4 * 3e38 + 2.0**-8 * 3e38}[kind]
    assert ((got.double() - x.double()).abs() <= step).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64])
def test_four_bits_up_to_the_largest_number_of_bf16(group):
    """Groups from -a to a, a up to the type's largest: 8 s is beyond fp32 from 0.94 of that on. Scale, middle and codes are those of the definition in 64
    bits; nothing reads back as NaN or infinity. (The largest, 15 s - a for s rounded up by up to 2^-9, stays below where bf16 rounds to infinity for
    these a.)"""
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    top = torch.finfo(torch.bfloat16).max
    a = torch.tensor([top, 3.35e38, 3.25e38, 3.2e38, 3.18e38, 1e38, 2.0**120, 2.0**119], dtype=torch.float64)
    x = (torch.linspace(-1, 1, group, dtype=torch.float64).repeat(64 // group)[None] * a[:, None]).to(torch.bfloat16).to(DEV)
    cache, used = empty_kv_quantized(1, 8, 1, 64, torch.uint8, group), torch.zeros(1, dtype=torch.int32, device=DEV)
    append_kv_quantized(None, x.view(1, 8, 1, 64), x.flip(-1).view(1, 8, 1, 64), *cache, used)
    got = read_kv_quantized(*cache, used, max_seqlen=8)
    done()
    for codes, scales, rows, values16 in ((cache[0], cache[2], x, got[0]), (cache[1], cache[3], x.flip(-1), got[1])):
        g = rows.double().cpu().unflatten(-1, (-1, group))
        low, high = g.amin(-1), g.amax(-1)
        s = ((high - low) / 15).float().to(torch.bfloat16)
        z = (low + 8 * s.double()).float().to(torch.bfloat16)
        assert torch.equal(bits(scales[0, :, 0]), bits(torch.stack([s, z], -1)))
        n = ((g - z.double()[..., None]) / s.double()[..., None]).round().clamp(-8, 7).flatten(-2) + 8
        kept = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[0, :, 0].cpu()
        assert ((kept.double() - n).abs() <= 1).all() and (kept == n).double().mean() > 0.95  # (ties, by products with 1 / s)
        assert values16.isfinite().all()
        step = s.double()[..., None] * (0.5 + 15 * 2.0**-8) * 1.01 + 2.0**-8 * high[..., None].abs() * 1.01  # as for special rows
        assert ((values16[0, :, 0].double().cpu().unflatten(-1, (-1, group)) - g).abs() <= step + 2.0**-8 * g.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,d,group", FORMS)
def test_reading_back(kind, d, group, dtype):
    """Padded and packed, every slot in its place, zeros elsewhere; values rounded once."""
    from flash_sparse_attn.utils.kvcache import read_kv_quantized

    eps, small = torch.finfo(dtype).eps, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for by_head, page, used in ((True, 0, [0, 1, 37, 40]), (False, 32, [64, 0, 33]), (True, 256, [700, 1])):
        b, hkv, cap = len(used), 3, 40
        g = torch.Generator().manual_seed(4)
        kw = {}
        if page:
            pool, table, _, _ = pages_for(g, used, 3, page)
            kw["page_table"] = table.to(DEV)
            cache = make_cache(2, pool, page, hkv, d, kind, group, by_head)
        else:
            cache = make_cache(2, b, cap, hkv, d, kind, group, by_head)
        want = []
        for codes, scales in ((cache[0], cache[2]), (cache[1], cache[3])):
            x = values(codes, scales)
            want.append([torch.stack([x[int(table[i, s // page]), s % page] if page else x[i, s] for s in range(n)]) if n else x[0, :0] for i, n in enumerate(used)])
        used_d = torch.tensor(used, dtype=torch.int32, device=DEV)
        most = max(used) + 5
        padded = read_kv_quantized(*cache, used_d, max_seqlen=most, dtype=dtype, **kw)
        # packed rows with a gap in front, sequences of other bounds than their lengths, rows behind the last
        cu = torch.tensor([2, *(2 + torch.tensor([n + 1 for n in used]).cumsum(0)).tolist()], dtype=torch.int32, device=DEV)
        total = int(cu[-1]) + 4
        packed = read_kv_quantized(*cache, used_d, cu_seqlens=cu, total=total, dtype=dtype, **kw)
        done()
        for pad, pack, rows in zip(padded, packed, want):
            full, flat = torch.zeros(pad.shape, dtype=torch.float64), torch.zeros(pack.shape, dtype=torch.float64)
            for i, r in enumerate(rows):
                full[i, :len(r)] = r
                flat[int(cu[i]):int(cu[i]) + len(r)] = r
            for got, ref in ((pad, full), (pack, flat)):
                # one fp32 rounding (4 bits: of the sum only, their product is exact) and one to 16 bits
                assert ((got.double().cpu() - ref).abs() <= (eps / 2 + 2.0**-23) * ref.abs() * 1.01 + small + 2.0**-22 * (kind == "int4")).all()
                assert not got[(ref == 0).all(-1).all(-1).to(DEV)].any()


@pytest.mark.gpu
def test_reading_into_buffers_and_bad_pages():
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import read_kv_quantized

    cache = make_cache(1, 5, 32, 2, 64, "int8")
    used, table = torch.tensor([40, 50], dtype=torch.int32, device=DEV), torch.tensor([[1, 2], [3, 0]], dtype=torch.int32, device=DEV)
    want = read_kv_quantized(*cache, used, page_table=table, max_seqlen=60)
    room = torch.full((2, 70, 4, 80), 7.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, :60, :2, 8:72], room[:, :60, 2:, 8:72]
    got = read_kv_quantized(*cache, used, page_table=table, max_seqlen=60, out=out)
    done()
    assert got[0] is out[0] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    room[:, :60, :, 8:72] = 7.0
    assert (room == 7.0).all()
    # all slots of a contiguous cache without lengths
    k, _ = read_kv_quantized(*cache, max_seqlen=32)
    assert torch.equal(k.double().cpu(), values(cache[0], cache[2]).to(torch.bfloat16).double())
    for bad in (-1, 5):
        table[1, 1] = bad
        k, v = read_kv_quantized(*cache, used, page_table=table, max_seqlen=60)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status 3"):
            fsa.check_status()
        assert torch.equal(k[0], want[0][0]) and torch.equal(k[1, :32], want[0][1, :32]) and not k[1, 32:].any() and not v[1, 32:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_a_captured_step_on_another_stream(kind):
    """Append and read captured on a side stream and replayed: lengths grow on the device, every replay stores the next row."""
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    cos, sin = tables(40, 32)
    q, k, v = normal(1, 3, 1, 4, 64), normal(2, 3, 1, 2, 64), normal(3, 3, 1, 2, 64)
    caches = [empty_kv_quantized(9, 32, 2, 64, KINDS[kind]) for _ in range(2)]
    used = [torch.tensor([30, 0, 31], dtype=torch.int32, device=DEV) for _ in range(2)]
    table = [torch.tensor([[4, -1], [-1, -1], [7, -1]], dtype=torch.int32, device=DEV) for _ in range(2)]
    free = torch.tensor([0, 1, 2, 3, 5], dtype=torch.int32, device=DEV)
    count = [torch.tensor([5], dtype=torch.int32, device=DEV) for _ in range(2)]

    def step(i):
        oq = append_kv_quantized(q, k, v, *caches[i], used[i], cos, sin, page_table=table[i], free_pages=free, free_count=count[i])
        return (oq,) + read_kv_quantized(*caches[i], used[i], page_table=table[i], max_seqlen=64)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = step(0)
        for n in range(4):
            with torch.no_grad():
                k.add_(0.25)
            graph.replay()
            want = step(1)
            side.synchronize()
            for a, b in zip(kept, want):
                assert torch.equal(a, b)
    done()
    assert used[0].tolist() == [34, 4, 35] and torch.equal(table[0], table[1]) and torch.equal(count[0], count[1])


@pytest.mark.gpu
def test_autograd_notices_what_was_written():
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized

    k = normal(1, 1, 1, 2, 64)
    cache = empty_kv_quantized(1, 9, 2, 64)
    used = torch.zeros(1, dtype=torch.int32, device=DEV)
    w = torch.ones(1, device=DEV).requires_grad_()
    y = (w * cache[2]).sum()
    append_kv_quantized(None, k, k, *cache, used)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        cache, used = empty_kv_quantized(1, 9, 2, 64), torch.zeros(1, dtype=torch.int32, device=DEV)
    append_kv_quantized(None, k, k, *cache, used)
    done()
    assert used.item() == 1


@pytest.mark.gpu
def test_axes_without_tables_or_positions_are_refused():
    """Both launchers: axes belong to tables and positions, neither goes without the others."""
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized

    cos, sin = tables(9, 32)
    k, ids = normal(1, 2, 1, 2, 64), torch.zeros(2, 2, 1, dtype=torch.int32, device=DEV)
    cache, used = empty_kv_quantized(2, 10, 2, 64), torch.zeros(2, dtype=torch.int32, device=DEV)
    append_kv_quantized(None, k, k, *cache, used, cos, sin, position_ids=ids, sections=[16, 16])  # (which a native launcher wants to have seen)
    done()
    assert used.tolist() == [1, 1]
    kept = [t.clone() for t in cache]
    for kw in (dict(sections=(16, 16)), dict(sections=[16, 16], position_ids=ids), dict(position_ids=ids), dict(cos=cos, sin=sin, sections=(16, 16)),
               dict(cos=cos, sin=sin, position_ids=ids), dict(sin=sin, sections=(16, 16), position_ids=ids), dict(cos=cos, sections=(16, 16), position_ids=ids)):
        with pytest.raises(AssertionError):
            append_kv_quantized(None, k, k, *cache, used, **kw)
    done()
    assert used.tolist() == [1, 1] and all(torch.equal(a, b) for a, b in zip(cache, kept))


def test_refusals_on_the_cpu():
    from flash_sparse_attn import _lib
    from flash_sparse_attn.utils import quantized_kvcache as m
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    bf, i32 = torch.bfloat16, torch.int32
    kc, vc, ks, vs = empty_kv_quantized(3, 32, 2, 64, device="cpu")
    k4, v4, ks4, vs4 = empty_kv_quantized(3, 32, 2, 64, torch.uint8, 32, device="cpu")
    assert kc.shape == (3, 32, 2, 64) and kc.stride() == (4096, 64, 2048, 1) and k4.shape == (3, 32, 2, 32) and ks4.shape == (3, 32, 2, 2, 2)
    for bad in (dict(dtype=torch.float16), dict(head_dim=24), dict(head_dim=144), dict(head_dim=96, dtype=torch.uint8), dict(dtype=torch.uint8, group_size=16)):
        with pytest.raises(AssertionError):
            empty_kv_quantized(**dict(dict(blocks=1, slots=1, heads_kv=1, head_dim=64, device="cpu"), **bad))
    table = torch.zeros(5, 2, dtype=i32)
    good = dict(key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, page_table=None, batch=3)
    four = dict(good, key_cache=k4, value_cache=v4, key_scales=ks4, value_scales=vs4)
    for ok in (good, four, dict(good, page_table=table, batch=5), dict(good, key_cache=torch.zeros(3, 32, 2, 64, dtype=torch.int8))):
        m.check_quantized_cache(**ok)
    flat = torch.zeros(3 * 32 * 2 * 64 + 1, dtype=torch.int8)
    for bad in (dict(batch=2), dict(value_cache=vc[:, :31]), dict(key_cache=kc.float()), dict(key_cache=kc.view(torch.uint8)), dict(value_cache=vc.view(torch.float8_e4m3fn)),
                dict(key_scales=ks[:, :31]), dict(key_scales=ks.half()), dict(key_scales=ks[..., 0]), dict(key_cache=kc[..., :24], value_cache=vc[..., :24]),
                dict(key_cache=flat[1:].view(3, 32, 2, 64)), dict(key_cache=kc[:1].expand(3, 32, 2, 64)), dict(key_scales=ks[:, :1].expand(3, 32, 2, 1)),
                dict(page_table=table.long(), batch=5), dict(page_table=table[:, 0], batch=5), dict(page_table=table[:1].expand(5, 2), batch=5),
                dict(key_cache=kc[:0], value_cache=vc[:0], key_scales=ks[:0], value_scales=vs[:0], batch=0),
                dict(key_scales=ks4, value_scales=vs4)):
        with pytest.raises(AssertionError):
            m.check_quantized_cache(**dict(good, **bad))
    for bad in (dict(key_scales=ks, value_scales=vs), dict(key_scales=ks4[..., :1], value_scales=vs4[..., :1]), dict(key_scales=ks4.half(), value_scales=vs4.half()),
                dict(key_scales=ks4.flip(-1).transpose(-1, -2)), dict(key_scales=ks4.repeat(1, 1, 1, 2, 1), value_scales=vs4.repeat(1, 1, 1, 2, 1)),
                dict(value_scales=vs4[..., :1, :])):
        with pytest.raises(AssertionError):
            m.check_quantized_cache(**dict(four, **bad))

    k, q, cos, sin = torch.zeros(3, 4, 2, 64, dtype=bf), torch.zeros(3, 4, 8, 64, dtype=bf), torch.zeros(9, 32), torch.zeros(9, 32)
    used, cu, ids = torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32), torch.zeros(2, 3, 4, dtype=i32)
    good = dict(query=q, key_new=k, value_new=k, key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, seqused_k=used, cos=cos, sin=sin, page_table=None,
                free_pages=None, free_count=None, cu_seqlens_new=None, seqlen_offsets=None, position_ids=None, sections=None, out=None)
    m._check_append(**good)
    m._check_append(**dict(good, query=None, cos=None, sin=None))
    m._check_append(**dict(good, position_ids=ids, sections=(16, 16)))
    m._check_append(**dict(good, query=q[0], key_new=k[0], value_new=k[0], cu_seqlens_new=cu))
    paged = dict(page_table=torch.zeros(3, 2, dtype=i32))
    m._check_append(**dict(good, **paged, free_pages=used, free_count=used[:1]))
    odd = torch.zeros(3 * 4 * 2 * 64 + 1, dtype=bf)[1:].view(3, 4, 2, 64)
    for bad in (dict(key_new=k.float(), value_new=k.float()), dict(value_new=k.half()), dict(value_new=k[:, :3]), dict(key_new=k[0], value_new=k[0]),
                dict(key_new=odd), dict(key_new=k[:2], value_new=k[:2]), dict(key_new=k[..., :1, :], value_new=k[..., :1, :]), dict(query=q[:, :, :7]),
                dict(query=q.half()), dict(query=q[:, :3]), dict(query=q[:, :, :0]), dict(cos=None), dict(cos=None, sin=None), dict(seqused_k=used.long()),
                dict(seqused_k=used[:2]), dict(cos=cos[:, :4], sin=sin[:, :4]), dict(cos=torch.zeros(9, 48), sin=torch.zeros(9, 48)),
                dict(cos=torch.zeros(9, 33)[:, :32], sin=torch.zeros(9, 33)[:, :32]), dict(position_ids=ids), dict(sections=(16, 16)),
                dict(position_ids=ids[:, :2], sections=(16, 16)), dict(position_ids=ids, sections=(16, 16), seqlen_offsets=3), dict(free_pages=used),
                dict(free_pages=used, free_count=used[:1]), dict(paged, free_count=used[:1]), dict(paged, free_pages=used.long(), free_count=used[:1]),
                dict(cu_seqlens_new=cu), dict(out=q[:, :3]), dict(out=q.half()), dict(query=None, out=q), dict(out=q[:1].expand(3, 4, 8, 64)),
                dict(query=None, cos=None, sin=None, seqlen_offsets=1)):
        with pytest.raises(AssertionError):
            m._check_append(**dict(good, **bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv_quantized(None, k, k, kc, vc, ks, vs, used)

    good = dict(key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, seqused_k=used, page_table=None, cu_seqlens=None, max_seqlen=7, total=None, dtype=bf,
                out=None)
    m._check_read(**good)
    m._check_read(**dict(good, cu_seqlens=cu, max_seqlen=None, total=9))
    room = torch.zeros(2, 3, 7, 2, 64, dtype=bf)
    m._check_read(**dict(good, out=tuple(room)))
    for bad in (dict(max_seqlen=None), dict(total=9), dict(cu_seqlens=cu), dict(cu_seqlens=cu, total=9), dict(dtype=torch.float32), dict(max_seqlen=-1),
                dict(seqused_k=used[:2]), dict(seqused_k=used.long()), dict(cu_seqlens=cu.long(), max_seqlen=None, total=9), dict(out=tuple(room[:, :2])),
                dict(cu_seqlens=cu[:1], max_seqlen=None, total=9), dict(out=tuple(room.half())), dict(out=(room[0], room[1][:1].expand(3, 7, 2, 64)))):
        with pytest.raises(AssertionError):
            m._check_read(**dict(good, **bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        read_kv_quantized(kc, vc, ks, vs, max_seqlen=3)
    lib = _lib.load()

    def call(args, fn, cache, kw):
        a = args()
        for n in ("k", "v", "k_scales", "v_scales"):
            setattr(a.cache, n, 256)
        a.cache.heads_kv, a.cache.head_dim, a.cache.capacity = 1, 64, 8
        a.batch, a.dtype, a.status = 1, _lib.DT_BF16, 256
        for n, _ in args._fields_:
            if n in ("k_new", "v_new", "seqused_k", "k_out", "v_out", "place_ws"):
                setattr(a, n, 256)
        for n, v in cache.items():
            setattr(a.cache, n, v)
        for n, v in kw.items():
            setattr(a, n, v)
        return getattr(lib, fn)(ctypes.byref(a), None)

    pages = dict(page_table=256, page_size=32, max_pages=1, num_pages=1)
    for args, fn, own in ((_lib.FsaKvAppendQuantArgs, "fsa_kv_append_quantized", dict(new_tokens=1)), (_lib.FsaKvReadQuantArgs, "fsa_kv_read_quantized", dict(seqlen=1))):
        for cache in (dict(k=None), dict(v_scales=None), dict(k=264), dict(k_scales=258), dict(heads_kv=0), dict(head_dim=0), dict(capacity=0), dict(k_stride_s=24),
                      dict(pages, page_size=0), dict(pages, max_pages=0), dict(pages, num_pages=0)):
            assert call(args, fn, cache, own) == -1, (fn, cache)
        for cache in (dict(format=3), dict(head_dim=72), dict(head_dim=144), dict(format=2, group=0), dict(format=2, group=16), dict(format=2, group=64, head_dim=96)):
            assert call(args, fn, cache, own) == -2, (fn, cache)
        assert call(args, fn, {}, dict(own, dtype=_lib.DT_F32)) == -2 and call(args, fn, {}, dict(own, batch=0)) == -1
        assert call(args, fn, {}, {}) == 0 and call(args, fn, {}, dict(own, status=None)) == -1
    turned = dict(new_tokens=1, cos=256, sin=256, rotary_dim=32, table_rows=1, table_dtype=_lib.DT_F32)
    for kw in (dict(k_new=None), dict(k_new=264), dict(k_stride_s=12), dict(heads_q=2), dict(turned, heads_q=2), dict(turned, cos=None), dict(turned, rotary_dim=80),
               dict(position_ids=256, axes=2), dict(turned, position_ids=256, axes=0), dict(turned, position_ids=256, axes=5), dict(free_pages=256, free_count=256)):
        assert call(_lib.FsaKvAppendQuantArgs, "fsa_kv_append_quantized", {}, dict(dict(new_tokens=1), **kw)) == -1, kw
    for kw in (dict(turned, rotary_dim=24), dict(turned, cos=260), dict(turned, table_stride=6)):
        assert call(_lib.FsaKvAppendQuantArgs, "fsa_kv_append_quantized", {}, kw) == -2, kw
    for kw in (dict(k_out=None), dict(v_out=264), dict(v_out_stride_h=4)):
        assert call(_lib.FsaKvReadQuantArgs, "fsa_kv_read_quantized", {}, dict(dict(seqlen=1), **kw)) == -1, kw
