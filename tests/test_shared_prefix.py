"""Decode over a prefix that the whole batch shares, against softmax attention over the concatenated keys in 64 bits: lengths from
none to long, group sizes, head sizes, pages, strides, rows without keys; and refusals."""

import ctypes

import pytest
import torch

from test_rotary import launcher  # noqa: F401

DEV = "cuda"


def normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


def reference(q, pk, pv, keys, values, scale=None):
    """q [B, Hq, D]; pk, pv [P, Hkv, D]; keys, values: one [n, Hkv, D] per sequence. Result, log-sum-exp, and sum |p v| (what is
    added up), on the GPU in 64 bits."""
    b, hq, d = q.shape
    hkv = pk.shape[1]
    scale = d**-0.5 if scale is None else scale
    out, lse, size = (torch.zeros(b, hq, n, dtype=torch.float64, device=q.device) for n in (d, 1, d))
    for i in range(b):
        k, v = torch.cat([pk, keys[i]]).double(), torch.cat([pv, values[i]]).double()
        if k.shape[0] == 0:
            lse[i] = -torch.inf
            continue
        s = torch.einsum("hgd,nhd->hgn", q[i].double().view(hkv, hq // hkv, d), k) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, d)
        size[i] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(hq, d)
        lse[i] = torch.logsumexp(s, -1).reshape(hq, 1)
    return out, lse[..., 0], size


def check(out, lse, want, q, pk, keys, scale=None):
    """Probabilities are rounded to 16 bits in front of the product (half a step, relative, of each term: at most eps / 2 of the
    terms' absolute sum) and the result once more (eps / 2 of it). Scores are sums of D products of exact 16-bit factors in fp32,
    off by less than D 2^-24 of the sum of their absolute values, A: that moves every probability by a fraction of at most
    2 D 2^-24 A scale (itself and the sum), the exponential and the sums by 2^-20 more, and the log-sum-exp by as much and the rounding of
    its own value. Probabilities below the type's normal values, relative to the largest, are off by half of its smallest step."""
    ref, ref_lse, size = want
    eps, d, hkv = torch.finfo(out.dtype).eps, q.shape[-1], pk.shape[1]
    scale = d**-0.5 if scale is None else scale
    reach = torch.cat([pk, *keys]).double().abs().amax(0) if pk.shape[0] + sum(k.shape[0] for k in keys) else torch.zeros_like(q[0, :hkv]).double()
    a = torch.einsum("bhgd,hd->bhg", q.double().abs().view(q.shape[0], hkv, -1, d), reach).reshape(q.shape[:2]) * scale
    f = 2 * d * 2.0**-24 * a + 2.0**-20
    tiny, count = torch.finfo(out.dtype).smallest_normal * eps / 2, pk.shape[0] + max(k.shape[0] for k in keys)
    bound = (eps / 2 + f[..., None]) * size + eps / 2 * ref.abs() * 1.01 + tiny * (1 + 6 * count)  # values below 6
    wrong = ~((out.double() - ref).abs() <= bound)
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}, worst {(out.double() - ref).abs()[wrong].max():.3g}"
    dead = ref_lse == -torch.inf
    assert torch.equal(lse == -torch.inf, dead) and not out[dead].any()
    assert ((lse.double() - ref_lse).abs()[~dead] <= (f + 2.0**-22 * ref_lse.abs())[~dead]).all()


def run(batch, prefix, lens, hq, hkv, d, dtype=torch.bfloat16, page=0, prefix_page=0, room=0, scale=None, spread=1.0,
        foreign=None, capacity=None, seed=0):
    """`room`: positions behind the prefix's end that exist but do not count; `foreign`: what lies in places that no key is in."""
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(seed)
    lens = [lens] * batch if isinstance(lens, int) else lens
    q = normal(g, batch, hq, d, dtype=dtype) * spread
    pk, pv = (normal(g, prefix, hkv, d, dtype=dtype) for _ in range(2))
    keys, values = ([normal(g, n, hkv, d, dtype=dtype) for n in lens] for _ in range(2))
    kw = dict(seqused_k=torch.tensor(lens, dtype=torch.int32, device=DEV), softmax_scale=scale)
    fill = 0.0 if foreign is None else foreign
    longest = max(lens) if capacity is None else capacity
    if page:
        slots = max(1, -(-longest // page))
        pool = batch * slots + 1
        perm = torch.randperm(pool, generator=g)
        table = perm[:batch * slots].view(batch, slots).to(torch.int32)
        k, v = (torch.full((pool, page, hkv, d), fill, dtype=dtype, device=DEV) for _ in range(2))
        for cache, rows in ((k, keys), (v, values)):
            for i in range(batch):
                for s in range(-(-lens[i] // page)):
                    part = rows[i][s * page:(s + 1) * page]
                    cache[int(table[i, s]), :part.shape[0]] = part
        kw["page_table"] = table.to(DEV)
    else:
        k, v = (torch.full((batch, longest, hkv, d), fill, dtype=dtype, device=DEV) for _ in range(2))
        for cache, rows in ((k, keys), (v, values)):
            for i in range(batch):
                cache[i, :lens[i]] = rows[i]
    if prefix_page:
        slots = -(-(prefix + room) // prefix_page)
        perm = torch.randperm(slots + 2, generator=g)
        cpk, cpv = (torch.full((slots + 2, prefix_page, hkv, d), fill, dtype=dtype, device=DEV) for _ in range(2))
        for cache, rows in ((cpk, pk), (cpv, pv)):
            for s in range(-(-prefix // prefix_page)):
                part = rows[s * prefix_page:(s + 1) * prefix_page]
                cache[int(perm[s]), :part.shape[0]] = part
        kw["prefix_page_table"] = perm[:slots].to(torch.int32).to(DEV)
    else:
        cpk, cpv = (torch.cat([t, torch.full((room, hkv, d), fill, dtype=dtype, device=DEV)]) for t in (pk, pv))
    if prefix_page or room:
        kw["prefix_seqused"] = torch.tensor([prefix], dtype=torch.int32, device=DEV)
    out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, cpk, cpv, return_lse=True, **kw)
    torch.cuda.synchronize()
    fsa.check_status()
    check(out, lse, reference(q, pk, pv, keys, values, scale), q, pk, keys, scale)
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_sizes(d, dtype):
    run(5, 300, [0, 1, 17, 64, 130], 8, 2, d, dtype)
    run(70, 700, 9, 8, 2, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [1, 2, 127, 128, 129, 255, 257, 1000, 5001, 20000])
def test_lengths_of_the_prefix(prefix):
    run(3, prefix, [1, 0, 33], 4, 1, 128)
    run(33, prefix, 3, 10, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,hq,hkv", [(1, 1, 1), (1, 8, 8), (127, 1, 1), (128, 1, 1), (129, 1, 1), (43, 6, 2), (43, 9, 3), (52, 5, 1),
                                          (64, 32, 8), (300, 4, 4), (17, 96, 1), (9, 65, 1), (7, 128, 2), (3, 300, 1), (2, 14, 2)])
def test_rows_and_groups(batch, hq, hkv):
    """One row to several query tiles, even and odd numbers of them, groups that end inside a tile."""
    run(batch, 901, [i % 7 for i in range(batch)], hq, hkv, 64)
    run(batch, 130, [i % 7 for i in range(batch)], hq, hkv, 128, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [8, 9, 12, 16, 31, 32, 33, 48, 63, 64, 65, 127, 129, 136])
def test_results_in_boxes_of_rows(group):
    """Pieces of a group's rows are written 32 rows and 32 columns at a time where there are more than eight: neighbours stay as they are."""
    run(23, 300, [(37 * i) % 400 for i in range(23)], 2 * group, 2, 80)
    run(90, 0, [1 + i % 3 for i in range(90)], 2 * group, 2, 48, torch.float16)
    run(3, 3000, [130, 0, 700], 2 * group, 2, 128)


@pytest.mark.gpu
def test_many_items_with_few_tiles():
    """More items than CTAs, one key tile each: shares that hold several items."""
    run(600, 100, 1, 32, 32, 64)
    run(600, 300, 1, 16, 16, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,prefix,own,hq,hkv", [(256, 4000, 4, 8, 2), (520, 20000, 1, 1, 1), (200, 2500, 199, 4, 1), (520, 3000, 300, 1, 1),
                                                     (600, 100, 1, 32, 32), (128, 700, 3000, 4, 2), (64, 1500, 3000, 8, 2), (130, 9000, 3, 16, 16)])
def test_shares(batch, prefix, own, hq, hkv):
    """Pairs of query tiles in equal pieces, one a CTA, with the own keys on the other CTAs, behind the pieces, and cut anywhere."""
    run(batch, prefix, [(97 * i) % (own + 1) for i in range(batch)], hq, hkv, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("page,prefix_page", [(0, 32), (32, 0), (32, 32), (64, 128), (128, 64), (256, 256)])
@pytest.mark.parametrize("prefix", [1, 31, 256, 1111])
def test_pages(page, prefix_page, prefix):
    run(6, prefix, [0, 1, 31, 32, 33, 300], 8, 2, 128, page=page, prefix_page=prefix_page)
    run(40, prefix, 40, 16, 4, 64, torch.float16, page=page, prefix_page=prefix_page, room=200)


@pytest.mark.gpu
@pytest.mark.parametrize("foreign", [float("nan"), float("inf"), -torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_behind_the_keys_does_not_matter(foreign, d):
    for page in (0, 64):
        run(5, 200, [0, 1, 17, 64, 100], 8, 2, d, page=page, prefix_page=page, room=100, foreign=foreign)
        run(150, 70, 5, 4, 2, d, page=page, prefix_page=page, room=300, foreign=foreign, capacity=40)


@pytest.mark.gpu
def test_rows_without_keys():
    out, lse = run(4, 0, [0, 3, 0, 200], 8, 2, 64)
    assert not out[0].any() and (lse[2] == -torch.inf).all()
    run(4, 0, 0, 8, 2, 128)
    run(4, 0, [0, 1, 2, 0], 8, 2, 128, page=32, prefix_page=32, room=100)
    run(4, 77, 0, 8, 2, 128)                       # a cache without positions
    run(130, 77, 0, 8, 2, 64, capacity=10)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [6.0, 40.0])
def test_concentrated_rows(spread):
    """Scores far apart: the running maximum moves in most tiles, and most probabilities vanish."""
    run(5, 2000, [0, 1, 17, 64, 500], 8, 2, 128, torch.float16, spread=spread)
    run(64, 1500, 30, 16, 4, 64, spread=spread)


@pytest.mark.gpu
def test_scales():
    for scale in (1e-6, 0.3, 1.0):
        run(5, 400, [0, 1, 17, 64, 500], 8, 2, 64, scale=scale)


@pytest.mark.gpu
def test_scores_of_minus_infinity():
    """Keys that score -inf with every row, in whole tiles at the front, weigh nothing; rows that see nothing else are 0."""
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(1)
    for batch in (3, 80):
        q = normal(g, batch, 4, 64).abs() + 0.1
        pk, pv = normal(g, 600, 2, 64), normal(g, 600, 2, 64)
        k, v = normal(g, batch, 9, 2, 64), normal(g, batch, 9, 2, 64)
        pk[:300] = -torch.inf
        out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk, pv, return_lse=True)
        kept = [k[i] for i in range(batch)], [v[i] for i in range(batch)]
        check(out, lse, reference(q, pk[300:], pv[300:], *kept), q, pk[300:], kept[0])
        out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk[:300], pv[:300], return_lse=True)
        check(out, lse, reference(q, pk[:0], pv[:0], *kept), q, pk[:0], kept[0])
        out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k[:, :0], v[:, :0], pk[:300], pv[:300], return_lse=True)
        assert not out.any() and (lse == -torch.inf).all()


@pytest.mark.gpu
def test_nan_stays_with_its_rows():
    """A NaN in a query, or in a key that counts, makes the rows that meet it NaN and no other, however the pieces are merged."""
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(2)
    for batch, prefix in ((3, 600), (3, 40_000), (80, 600), (500, 600)):
        q = normal(g, batch, 4, 64)
        pk, pv = normal(g, prefix, 2, 64), normal(g, prefix, 2, 64)
        k, v = normal(g, batch, 9, 2, 64), normal(g, batch, 9, 2, 64)
        clean, clean_lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk, pv, return_lse=True)
        for where in ("query", "own key", "prefix key"):
            q1, k1, pk1, hit = q.clone(), k.clone(), pk.clone(), torch.zeros(batch, 4, dtype=torch.bool, device=DEV)
            if where == "query":
                q1[1, 2, 5], hit[1, 2] = torch.nan, True
            elif where == "own key":
                k1[2, 8, 1, 3], hit[2, 2:] = torch.nan, True
            else:
                pk1[prefix - 1, 0, 63], hit[:, :2] = torch.nan, True
            out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q1, k1, v, pk1, pv, return_lse=True)
            assert out[hit].isnan().all() and lse[hit].isnan().all(), where
            assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit]), where


@pytest.mark.gpu
def test_strides_buffers_streams_and_graphs():
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(2)
    b, hq, hkv, d, n, p = 21, 12, 4, 64, 70, 333
    q = normal(g, b, hq * 2, d + 8)[:, ::2, :d]
    k, v = (normal(g, b, hkv, n, d).transpose(1, 2) for _ in range(2))
    both = normal(g, 2, hkv, p, d + 16)
    pk, pv = both[0, ..., :d].transpose(0, 1), both[1, ..., 16:].transpose(0, 1)
    buf, lse_buf = torch.zeros(b, hq, 2 * d, dtype=torch.bfloat16, device=DEV), torch.zeros(b, hq, device=DEV)
    used = torch.arange(b, dtype=torch.int32, device=DEV) * 3
    length = torch.tensor([p], dtype=torch.int32, device=DEV)

    def call(**kw):
        return fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk, pv, seqused_k=used, prefix_seqused=length, return_lse=True, **kw)

    out, lse = call(out=buf[..., :d], lse=lse_buf)
    assert out.data_ptr() == buf.data_ptr() and lse is lse_buf and not buf[..., d:].any()

    def expect(out, lse, n_prefix):
        lens = used.tolist()
        keys, values = [k[i, :lens[i]] for i in range(b)], [v[i, :lens[i]] for i in range(b)]
        check(out, lse, reference(q, pk[:n_prefix], pv[:n_prefix], keys, values), q, pk[:n_prefix], keys)

    expect(out, lse, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, out) and torch.equal(l2, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, l3 = call()
    for n_prefix, shift in ((p, 0), (p - 200, 5), (0, 1), (1, 0), (p, 7)):  # lengths live on the device
        length.fill_(n_prefix)
        used.add_(shift).clamp_(max=n)
        graph.replay()
        torch.cuda.synchronize()
        expect(o3, l3, n_prefix)
    fsa.check_status()


@pytest.mark.gpu
def test_equals_the_plain_decode_and_repeats():
    """The same keys as one cache through flash_dense_attn_with_kvcache_func, and run-to-run equality."""
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(3)
    b, hq, hkv, d, p, n = 24, 16, 4, 128, 1000, 90
    q, pk, pv = normal(g, b, hq, d), normal(g, p, hkv, d), normal(g, p, hkv, d)
    k, v = normal(g, b, n, hkv, d), normal(g, b, n, hkv, d)
    out = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk, pv)
    assert torch.equal(out, fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pk, pv))
    whole = [torch.cat([a.expand(b, -1, -1, -1), c], 1).contiguous() for a, c in ((pk, k), (pv, v))]
    plain = fsa.flash_dense_attn_with_kvcache_func(q, *whole)
    assert (out.float() - plain.float()).abs().max() < 2e-2  # two results off by up to 2^-8 of terms that add up to about 0.8


@pytest.mark.gpu
def test_a_cache_longer_than_32_bits():
    """The prefix's last pages lie 4.4e9 elements into the pool."""
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(4)
    pages, page, hkv, d = 17000, 256, 8, 128
    k = torch.zeros(pages, page, hkv, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    rows = normal(g, 2, 2 * page, hkv, d)
    k[-2:], v[-2:] = rows[0].view(2, page, hkv, d), rows[1].view(2, page, hkv, d)
    q = normal(g, 3, 16, d)
    table = torch.tensor([[pages - 1], [pages - 2], [0]], dtype=torch.int32, device=DEV)
    used = torch.tensor([256, 100, 0], dtype=torch.int32, device=DEV)
    common = torch.tensor([pages - 2, pages - 1], dtype=torch.int32, device=DEV)
    out, lse = fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, k, v, page_table=table, seqused_k=used, prefix_page_table=common, return_lse=True)
    keys = [rows[0, page:], rows[0, :100], rows[0, :0]]
    values = [rows[1, page:], rows[1, :100], rows[1, :0]]
    check(out, lse, reference(q, rows[0], rows[1], keys, values), q, rows[0], keys)
    fsa.check_status()


@pytest.mark.gpu
def test_a_prefix_page_outside_the_pool_is_reported():
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(5)
    q, k, v = normal(g, 2, 4, 64), normal(g, 2, 8, 2, 64), normal(g, 2, 8, 2, 64)
    pool = normal(g, 3, 32, 2, 64)
    for bad in (-1, 3, 1 << 30):
        table = torch.tensor([0, bad, 1, 12345], dtype=torch.int32, device=DEV)
        used = torch.tensor([96], dtype=torch.int32, device=DEV)  # the last entry holds no key
        fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pool, pool, prefix_page_table=table, prefix_seqused=used)
        with pytest.raises(RuntimeError, match="device status 3"):
            fsa.check_status()
    table[1] = 2
    fsa.flash_dense_attn_with_shared_prefix_func(q, k, v, pool, pool, prefix_page_table=table, prefix_seqused=used)
    fsa.check_status()


@pytest.mark.gpu
def test_a_serving_step():
    """Prompt into pages, then steps of one token: rotated append behind the prefix, decode over prefix and own pages."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_rotary
    from test_rotary import tables, turn

    g = torch.Generator().manual_seed(6)
    b, hq, hkv, d, page, p, slots = 9, 8, 2, 128, 64, 150, 2
    pool = 3 + b * slots
    kc, vc = (torch.zeros(pool, page, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cos, sin = tables(400, d // 2)
    free, count = torch.arange(pool, dtype=torch.int32, device=DEV), torch.tensor([pool], dtype=torch.int32, device=DEV)
    common, length = torch.full((1, 3), -1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    prompt = normal(g, 2, 1, p, hkv, d)
    append_kv_rotary(None, prompt[0], prompt[1], kc, vc, length, cos, sin, page_table=common, free_pages=free, free_count=count)
    table, used = torch.full((b, slots), -1, dtype=torch.int32, device=DEV), torch.zeros(b, dtype=torch.int32, device=DEV)
    steps = 70
    q, k, v = normal(g, steps, b, 1, hq, d), normal(g, steps, b, 1, hkv, d), normal(g, steps, b, 1, hkv, d)
    for t in range(steps):
        turned = append_kv_rotary(q[t], k[t], v[t], kc, vc, used, cos, sin, page_table=table, free_pages=free, free_count=count, seqlen_offsets=length.expand(b).contiguous())
        out, lse = fsa.flash_dense_attn_with_shared_prefix_func(turned[:, 0], kc, vc, kc, vc, page_table=table, seqused_k=used,
                                                                prefix_page_table=common[0], prefix_seqused=length, return_lse=True)
    fsa.check_status()
    assert used.tolist() == [steps] * b and int(length) == p
    # keys as they are stored (16 bits); the rotation has its own tests
    store = lambda x, at: turn(x, cos[at], sin[at], False)[0].to(torch.bfloat16).to(DEV)  # noqa: E731
    pk = store(prompt[0, 0], torch.arange(p))
    keys = [store(k[:, i, 0], torch.arange(steps) + p) for i in range(b)]
    last = store(q[-1, :, 0], torch.full((b,), p + steps - 1))
    want = reference(last, pk, prompt[1, 0], keys, [v[:, i, 0] for i in range(b)])
    # roundings of ties may differ between the two rotations: one step of some key elements, 2^-8 of them, moves a score little
    assert (out.double() - want[0]).abs().max() < 2e-2 and (lse.double() - want[1]).abs().max() < 2e-2


def test_refusals():
    from flash_sparse_attn import _lib
    from flash_sparse_attn.ops.triton import flash_prefix
    from flash_sparse_attn.ops.triton.interface import flash_dense_attn_with_shared_prefix_func

    bf, i32 = torch.bfloat16, torch.int32
    q, k, pk = torch.zeros(3, 8, 64, dtype=bf), torch.zeros(3, 32, 2, 64, dtype=bf), torch.zeros(9, 2, 64, dtype=bf)
    good = dict(query=q, key=k, value=k, prefix_key=pk, prefix_value=pk, softmax_scale=None, page_table=None, seqused_k=None,
                prefix_page_table=None, prefix_seqused=None, out=None, lse=None)
    table, pages = torch.zeros(3, 4, dtype=i32), torch.zeros(5, 32, 2, 64, dtype=bf)
    flash_prefix._check(**good)
    flash_prefix._check(**dict(good, key=pages, value=pages, page_table=table, prefix_key=pages, prefix_value=pages, prefix_page_table=table[0]))
    for bad in (dict(query=q[0]), dict(query=q.half()), dict(query=q[:, :7]), dict(query=q[:2]), dict(query=q[..., :32]), dict(value=k[:, :31]),
                dict(query=q.float(), key=k.float(), value=k.float(), prefix_key=pk.float(), prefix_value=pk.float()),
                dict(prefix_value=pk[:8]), dict(prefix_key=pk.half(), prefix_value=pk.half()), dict(prefix_key=pk[None], prefix_value=pk[None]),
                dict(prefix_key=pk[:, :1], prefix_value=pk[:, :1]), dict(value=k[..., None, :, 0]),
                dict(prefix_page_table=table[0]), dict(prefix_key=pages[:, :20], prefix_value=pages[:, :20], prefix_page_table=table[0]),
                dict(prefix_key=pages, prefix_value=pages, prefix_page_table=table), dict(page_table=table[:2], key=pages, value=pages),
                dict(prefix_key=pages, prefix_value=pages, prefix_page_table=table[0].long()), dict(key=pages, value=pages, page_table=table.long()),
                dict(seqused_k=torch.zeros(3)), dict(seqused_k=torch.zeros(2, dtype=i32)), dict(prefix_seqused=torch.zeros(2, dtype=i32)),
                dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")), dict(out=q[:2]), dict(out=q.half()),
                dict(lse=torch.zeros(3, 8, dtype=bf)), dict(query=torch.zeros(3 * 8 * 64 + 1, dtype=bf)[1:].view(3, 8, 64)),
                dict(query=q[:, :, :24], key=k[..., :24], value=k[..., :24], prefix_key=pk[..., :24], prefix_value=pk[..., :24]),
                dict(query=q.repeat(1, 1, 3), key=k.repeat(1, 1, 1, 3), value=k.repeat(1, 1, 1, 3), prefix_key=pk.repeat(1, 1, 3), prefix_value=pk.repeat(1, 1, 3))):
        with pytest.raises(AssertionError):
            flash_prefix._check(**dict(good, **bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        flash_dense_attn_with_shared_prefix_func(q, k, k, pk, pk)
    lib = _lib.load()

    def call(**kw):
        a = _lib.FsaSharedPrefixArgs()
        for n in ("q", "k", "v", "prefix_k", "prefix_v", "out", "lse", "status", "out_partial", "sum_partial", "plan_ws"):
            setattr(a, n, 256)
        a.batch, a.heads_q, a.heads_kv, a.head_dim, a.seqlen_k, a.prefix_seqlen, a.softmax_scale = 2, 4, 1, 64, 10, 10, 1.0
        a.k_stride_s = a.v_stride_s = a.prefix_k_stride_s = a.prefix_v_stride_s = 64
        a.k_stride_b = a.v_stride_b = 640
        a.dtype = _lib.DT_BF16
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.fsa_decode_shared_prefix(ctypes.byref(a), None)

    pages = dict(page_table=256, page_size=64, max_pages=1, num_pages=1)
    common = dict(prefix_page_table=256, prefix_page_size=64, prefix_max_pages=1, prefix_num_pages=1)
    for kw in (dict(q=None), dict(out=None), dict(lse=None), dict(status=None), dict(plan_ws=None), dict(out_partial=None), dict(out_partial=260), dict(plan_ws=260),
               dict(k=None), dict(prefix_v=None), dict(seqlen_k=-1), dict(prefix_seqlen=-1), dict(batch=0), dict(heads_kv=3), dict(head_dim=136),
               dict(head_dim=60), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(out=257),
               dict(out=258), dict(o_stride_b=3), dict(q=264), dict(q_stride_b=4), dict(q_stride_h=4), dict(pages, page_size=48),
               dict(pages, max_pages=-1), dict(common, prefix_page_size=16), dict(common, prefix_num_pages=-1), dict(pages, max_pages=1 << 25)):
        assert call(**kw) == -1, kw
    assert call(dtype=_lib.DT_E4M3) == -2 and call(batch=1 << 29, heads_q=4, heads_kv=1) == -2


def test_argument_blocks_match_the_header():
    import os
    import re

    from flash_sparse_attn import _lib

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fsa_b200.h")).read()
    for name in ("FsaSharedPrefixArgs", "FsaSharedPrefixWorkspace"):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1), flags=re.S)
        fields = [re.findall(r"[A-Za-z_]\w*", part)[-1] for stmt in body.split(";") if stmt.strip() for part in stmt.split(",")]
        assert fields == [f[0] for f in getattr(_lib, name)._fields_]


def test_expanded_result_buffers_are_refused():
    """Rows on top of one another: which of them stays would be chance."""
    from flash_sparse_attn.ops.triton import flash_prefix

    q, k, pk = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((3, 8, 64), (3, 32, 2, 64), (9, 2, 64)))
    good = dict(query=q, key=k, value=k, prefix_key=pk, prefix_value=pk, softmax_scale=None, page_table=None, seqused_k=None,
                prefix_page_table=None, prefix_seqused=None, out=None, lse=None)
    flash_prefix._check(**dict(good, out=torch.zeros(3, 16, 64, dtype=torch.bfloat16)[:, ::2], lse=torch.zeros(3, 20)[:, :8]))
    flash_prefix._check(**dict(good, query=q[:1], key=k[:1], value=k[:1], out=q[:1].expand(1, 8, 64)))
    for bad in (dict(out=q[:1].expand(3, 8, 64)), dict(out=q[:, :1].expand(3, 8, 64)), dict(lse=torch.zeros(1, 8).expand(3, 8))):
        with pytest.raises(AssertionError):
            flash_prefix._check(**dict(good, **bad))


@pytest.mark.gpu
def test_expanded_result_buffers_are_refused_by_the_call():
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(7)
    q, k, pk = normal(g, 3, 8, 64), normal(g, 3, 32, 2, 64), normal(g, 9, 2, 64)
    for bad in (dict(out=q[:1].clone().expand(3, 8, 64)), dict(out=q[:, :1].clone().expand(3, 8, 64)),
                dict(lse=torch.zeros(1, 8, device=DEV).expand(3, 8))):
        with pytest.raises(AssertionError):
            fsa.flash_dense_attn_with_shared_prefix_func(q, k, k, pk, pk, **bad)
