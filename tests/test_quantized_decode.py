"""Decode over a cache whose rows carry their own scales, against softmax attention over the values in 64 bits: formats, head sizes and
groups, lengths from none to long, pages, chosen positions, the ways that work is shared out, special values, other streams and
captured calls; a serving loop of append, read and decode; and refusals."""

import ctypes

import pytest
import torch

from test_quantized_kvcache import KINDS, make_cache, values
from test_rotary import done, launcher, normal, tables  # noqa: F401

DEV = "cuda"
TOP = {"int8": 127, "e4m3": 448, "int4": 8}


def reference(q, keys, vals, scale):
    """q [B, Hq, D]; keys, vals: one [n, Hkv, D] per sequence in 64 bits. Result, log-sum-exp and sum |p v|, worked out where the queries are."""
    b, hq, d = q.shape
    out, lse, size = (torch.zeros(b, hq, n, dtype=torch.float64, device=q.device) for n in (d, 1, d))
    lse -= torch.inf
    for i in range(b):
        if keys[i].shape[0] == 0:
            continue
        k, v = (x.permute(1, 0, 2).to(q.device) for x in (keys[i], vals[i]))  # [Hkv, n, D]
        s = q[i].double().view(k.shape[0], -1, d) @ k.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        out[i], size[i] = (torch.matmul(p, x).reshape(hq, d) for x in (v, v.abs()))
        lse[i] = torch.logsumexp(s, -1).reshape(hq, 1)
    return out.cpu(), lse[..., 0].cpu(), size.cpu()


def check(out, lse, q, keys, vals, reach_k, reach_v, scale=None):
    """Scores are sums of D products of exact factors in fp32, off by less than D 2^-24 of the sum of their absolute values A (of 4 bits:
    `reach` counts code and centre apart), and by 2^-24 of largest |q| times sum |k| for the bits that small elements of a row of queries lose
    as fp16; that moves a probability by twice as much, the exponential and the joining of parts by 2^-19 more. A probability times a scale is
    rounded to fp16: 2^-11 of the term, or 2^-25 of the largest value that a code can stand for; the result once more."""
    b, hq, d = q.shape
    scale = d**-0.5 if scale is None else scale
    ref, ref_lse, size = reference(q, keys, vals, scale)
    qa = q.double().cpu().abs().view(b, -1, hq // reach_k.shape[0] if reach_k.shape[0] else 1, d)
    a = torch.einsum("bhgd,hd->bhg", qa, reach_k).reshape(b, hq) * scale
    loss = (qa.amax(-1) * reach_k.sum(-1)[None, :, None]).reshape(b, hq) * scale * 2.0**-24
    f = 2 * (d * 2.0**-24 * a + loss) + 2.0**-19
    eps, count = torch.finfo(out.dtype).eps, max(k.shape[0] for k in keys)
    most = reach_v.max()
    bound = (2.0**-11 + f)[..., None] * torch.maximum(size, size.new_tensor(0)) + eps / 2 * ref.abs() * 1.01 + count * 2.0**-25 * most + 2.0**-20 * most
    bound = bound + torch.finfo(out.dtype).smallest_normal * eps
    got = out.double().cpu()
    wrong = ~((got - ref).abs() <= bound)
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}, worst {(got - ref).abs()[wrong].max():.3g} of {bound[wrong].min():.3g}"
    dead = ref_lse == -torch.inf
    lse = lse.double().cpu()
    assert torch.equal(lse == -torch.inf, dead) and not got[dead].any()
    assert ((lse - ref_lse).abs()[~dead] <= (f + 2.0**-21 * ref_lse.abs())[~dead]).all()


def run(lens, hq, hkv, d, kind="int8", group=64, dtype=torch.bfloat16, page=0, by_head=True, topk=0, scale=None, spread=1.0, capacity=None, seed=0, poison=False,
        twice=True):
    import flash_sparse_attn as fsa

    g = torch.Generator().manual_seed(seed)
    b, cap = len(lens), max(max(lens), 1) if capacity is None else capacity
    q = normal(seed + 1, b, hq, d, dtype=dtype) * spread
    kw = dict(seqused_k=torch.tensor(lens, dtype=torch.int32, device=DEV), softmax_scale=scale)
    if page:
        slots = -(-cap // page)
        pool = b * slots + 2
        table = torch.randperm(pool, generator=g)[:b * slots].view(b, slots).to(torch.int32)
        kw["page_table"] = table.to(DEV)
        cache = make_cache(seed + 2, pool, page, hkv, d, kind, group, by_head)
    else:
        table = None
        cache = make_cache(seed + 2, b, cap, hkv, d, kind, group, by_head)
    all_k, all_v = values(cache[0], cache[2]), values(cache[1], cache[3])

    def rows(x, i, n):
        return x[table[i, :-(-n // page)].long()].flatten(0, 1)[:n] if page else x[i, :n]

    keys, vals = ([rows(x, i, n) for i, n in enumerate(lens)] for x in (all_k, all_v))
    if topk:
        at = torch.randint(-3, cap + 3, (b, topk), generator=g).to(torch.int32)  # entries outside are left out, the same one may stand twice
        kw["gather_kv_indices"] = at.to(DEV)
        pick = [a[(a >= 0) & (a < n)].long() for a, n in zip(at, lens)]
        keys, vals = [k[p] for k, p in zip(keys, pick)], [v[p] for v, p in zip(vals, pick)]
    # the sizes of what is added up: of 4 bits codes and centres apart
    def reach(codes, scales, x):
        if kind != "int4":
            return x.abs().amax((0, 1))
        s, z = scales.double().cpu()[..., :1].abs(), scales.double().cpu()[..., 1:].abs()
        return (8 * s + z).expand(*s.shape[:-1], d // s.shape[-2]).flatten(-2).amax((0, 1))

    reach_k, reach_v = reach(cache[0], cache[2], all_k), reach(cache[1], cache[3], all_v)
    if poison:  # what lies behind the last position, and in pages of nobody
        inside = torch.zeros(cache[0].shape[:2], dtype=torch.bool)
        for i, n in enumerate(lens):
            for s in range(n):
                inside[(int(table[i, s // page]), s % page) if page else (i, s)] = True
        for t in cache:
            (t if t.dtype.is_floating_point and t.dtype != torch.float8_e4m3fn else t.view(torch.uint8))[~inside.to(DEV)] = float("nan") if t.dtype in (
                torch.float32, torch.bfloat16) else 255
    out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache, return_lse=True, **kw)
    if twice:  # no order of arrival in it
        again = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache, return_lse=True, **kw)
    done()
    if twice:
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    check(out, lse, q, keys, vals, reach_k, reach_v, scale)
    return out, lse


FORMS = [("int8", 128, 64), ("int8", 96, 64), ("int8", 64, 64), ("int8", 48, 64), ("int8", 16, 64), ("e4m3", 128, 64), ("e4m3", 80, 64), ("e4m3", 32, 64),
         ("int4", 128, 64), ("int4", 128, 32), ("int4", 96, 32), ("int4", 64, 64), ("int4", 64, 32), ("int4", 32, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,d,group", FORMS)
def test_formats_and_head_sizes(kind, d, group, dtype):
    kw = dict(kind=kind, d=d, group=group, dtype=dtype)
    run([0, 1, 15, 16, 17, 250], 8, 2, **kw)
    run([700, 3, 1300], 10, 1, page=64, by_head=False, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (8, 1), (9, 1), (16, 1), (17, 1), (40, 1), (35, 5), (14, 7), (64, 8)])
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_groups_of_heads(kind, hq, hkv):
    run([33, 1, 200], hq, hkv, 64, kind)
    run([500], hq, hkv, 128, kind, page=32)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 16, 31, 100, 1000, 2001, 20000, 70001])
@pytest.mark.parametrize("kind,d", [("int8", 128), ("int4", 128), ("e4m3", 64)])
def test_lengths(kind, d, n):
    """From a warp's tile to pieces of one item in every CTA."""
    run([n], 4, 1, d, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
def test_ways_that_work_is_shared_out(kind):
    run([5] * 300, 8, 2, 64, kind)                          # many items a warp
    run([40, 0, 0, 3000, 1, 0, 17] * 9, 8, 2, 128, kind)    # short and long side by side
    run([0] * 7, 8, 2, 128, kind)                           # nothing
    run([100] * 2000, 2, 1, 64, kind, twice=False)          # more sequences than lanes, many each
    run([9000, 4] + [0] * 30, 4, 4, 64, kind, page=256)
    run([(7 * i) % 41 for i in range(1500)], 1, 1, 64, kind, twice=False)  # lengths read side by side
    run([0] * 300 + [6000] + [0] * 33, 2, 1, 64, kind)      # one among many without a key
    run([3], 4, 1, 64, kind, capacity=5000)                 # room for more than there is


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d", [("int8", 128), ("int4", 64)])
@pytest.mark.parametrize("batch,hkv,per", [(1, 13, 4), (3, 5, 4), (16, 2, 1), (33, 1, 12), (69, 1, 4), (35, 2, 4), (148, 1, 4), (149, 1, 4)])
def test_few_tiles_and_many_sequences(kind, d, batch, hkv, per):
    """Items that a cluster of 8, 4, 2 or 1 takes, or the list; lengths from none up to what a cluster is given (4 tiles a warp of 8 to 12), and past it."""
    rng = torch.Generator().manual_seed(batch)
    for capacity in (40, 1290, 3100):
        lens = [capacity, *torch.randint(0, capacity + 1, (batch - 1,), generator=rng).tolist()]
        lens[batch // 2] = 0 if batch > 1 else capacity
        run(lens, hkv * per, hkv, d, kind, twice=False)
    run([700] * batch, hkv * per, hkv, d, kind, page=64, topk=500, twice=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
@pytest.mark.parametrize("page", [0, 32, 64, 128, 256])
def test_pages_and_what_lies_behind_the_last_position(kind, group, page):
    run([0, 1, 31, 32, 33, 300, 255], 8, 2, 128, kind, group, page=page, poison=True, capacity=320)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("topk", [1, 16, 37, 400])
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
def test_chosen_positions(kind, topk, page):
    run([0, 1, 50, 900, 333], 8, 2, 128, kind, page=page, topk=topk, capacity=960)
    run([5000, 4000], 12, 1, 64, kind, page=page, topk=topk)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
@pytest.mark.parametrize("spread", [1e-6, 30.0, 1e20])
def test_size_of_queries(kind, spread):
    """bf16 queries far outside what fp16 holds."""
    run([200, 30], 8, 2, 128, kind, spread=spread, scale=0.1 / spread)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
@pytest.mark.parametrize("factor", [1e-20, 1e-3, 1e6, 1e18])
def test_size_of_values(kind, factor):
    """Value scales far outside what fp16 holds, and growing along a sequence. The result follows the values' size."""
    import flash_sparse_attn as fsa

    q = normal(1, 2, 4, 64)
    k, v, ks, vs = make_cache(3, 2, 400, 2, 64, kind)
    used = torch.tensor([400, 37], dtype=torch.int32, device=DEV)
    one = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, seqused_k=used)
    exponent = torch.tensor(factor).log2().round()  # a power of two: the same numbers in other units
    two = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, (vs.float() * 2.0**exponent.item()).to(vs.dtype), seqused_k=used)
    done()
    assert torch.equal(one.float(), two.float() * 2.0**-exponent.item())
    grow = torch.linspace(0, 30, 400, device=DEV).round().exp2().view((1, 400) + (1,) * (vs.ndim - 2))
    vs = (vs.float() * grow).to(vs.dtype)
    out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, seqused_k=used, return_lse=True)
    done()
    vals, keys = values(v, vs), values(k, ks)
    ref, _, size = reference(q, [keys[i, :n] for i, n in enumerate(used.tolist())], [vals[i, :n] for i, n in enumerate(used.tolist())], 0.125)
    # as in check(); the largest terms are 2^30 times the first
    assert ((out.double().cpu() - ref).abs() <= (2.0**-8 + 2.0**-10) * size.amax(-1, keepdim=True)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
def test_log_sum_exps_of_few_keys_are_fp32(kind, group):
    """The root mean square of what 2400 of them are off by: four roundings of 2^-24 (row scales, softmax scale, exponentials' sum, its logarithm) of
    their own size, and the sum over columns, which the matrix instruction takes sixteen at a time: 2^-22 in all."""
    import flash_sparse_attn as fsa

    q, (k, v, ks, vs) = normal(1, 300, 8, 64), make_cache(2, 300, 2, 2, 64, kind, group)
    _, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, return_lse=True)
    done()
    want = reference(q, list(values(k, ks)), list(values(v, vs)), 0.125)[1]
    assert (lse.double().cpu() - want).norm() <= 2.0**-22 * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
def test_values_near_the_top_of_bf16(kind):
    """Values around 2^113: the same numbers as small ones in other units."""
    import flash_sparse_attn as fsa

    q = normal(1, 2, 4, 64)
    k, v, ks, vs = make_cache(3, 2, 70, 2, 64, kind)
    one = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs)
    two = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, (vs.float() * 2.0**112).to(vs.dtype))
    done()
    assert two.abs().max() > 2.0**110 and torch.equal(one.float(), two.float() * 2.0**-112)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4", "e4m3"])
def test_infinities_and_nan_stay_in_their_row(kind):
    """A stored row that stands for NaN makes the results of the sequence that attends to it NaN, and no others."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized

    for what in ("key", "value"):
        cache = empty_kv_quantized(3, 600, 1, 64, KINDS[kind])
        used = torch.zeros(3, dtype=torch.int32, device=DEV)
        k, v = normal(1, 3, 500, 1, 64), normal(2, 3, 500, 1, 64)
        (k if what == "key" else v)[1, 321, 0, 5] = float("inf")
        append_kv_quantized(None, k, v, *cache, used)
        q = normal(3, 3, 4, 64)
        out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache, seqused_k=used, return_lse=True)
        done()
        assert out[1].isnan().any(-1).all() and not out[0].isnan().any() and not out[2].isnan().any()
        assert bool(lse[1].isnan().all()) == (what == "key") and lse[0].isfinite().all()
        q[2, 1] = float("nan")
        out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache, seqused_k=used, return_lse=True)
        done()
        assert out[2, 1].isnan().all() and not out[2, 0].isnan().any() and not out[2, 2:].isnan().any() and lse[2, 1].isnan()


@pytest.mark.gpu
def test_growing_maxima_and_one_outlier():
    """Scores that rise along the sequence move the reference maximum again and again; one key far above the rest takes it all."""
    import flash_sparse_attn as fsa

    q = torch.ones(1, 8, 64, dtype=torch.bfloat16, device=DEV)
    k, v, ks, vs = make_cache(3, 1, 3000, 1, 64, "int8")
    k.fill_(100)
    ks[0, :, 0, 0] = torch.linspace(-0.05, 0.05, 3000, device=DEV)
    keys, vals = values(k, ks)[0], values(v, vs)[0]
    out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, return_lse=True)
    done()
    check(out, lse, q, [keys], [vals], keys.abs().amax(0), vals.abs().amax(0))
    ks[0, 1234] = 1.0
    out = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs)
    done()
    assert torch.equal(out[0].float().cpu(), vals[1234].expand(8, 64).to(torch.bfloat16).float())


@pytest.mark.gpu
def test_pages_outside_the_pool():
    import flash_sparse_attn as fsa

    k, v, ks, vs = make_cache(1, 6, 32, 2, 64, "int8")
    q, used = normal(2, 2, 8, 64), torch.tensor([90, 64], dtype=torch.int32, device=DEV)
    table = torch.tensor([[0, 1, 2], [3, 4, 99]], dtype=torch.int32, device=DEV)  # the last one holds no key
    want = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, page_table=table, seqused_k=used)
    done()
    at = torch.arange(100, dtype=torch.int32, device=DEV).expand(2, 100).contiguous()
    for bad in (-1, 6):
        for kw in ({}, dict(gather_kv_indices=at)):
            table[0, 1] = bad
            out = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, page_table=table, seqused_k=used, **kw)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="status 3"):
                fsa.check_status()
            assert (out[1].float() - want[1].float()).abs().max() < 2.0**-6 and out[0].isfinite().all()


@pytest.mark.gpu
def test_strides_buffers_and_single_dimensions():
    import flash_sparse_attn as fsa

    k, v, ks, vs = make_cache(1, 3, 64, 2, 64, "int8")
    q = normal(2, 3, 8, 64)
    want, want_lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, return_lse=True)
    wide = torch.zeros(3, 64, 5, 160, dtype=torch.int8, device=DEV)
    k2, v2 = wide[:, :, 1:3, 16:80], wide[:, :, 3:5, 80:144]
    k2.copy_(k), v2.copy_(v)
    scales = torch.zeros(2, 3, 64, 2, 3, device=DEV)
    scales[0, ..., 1:2], scales[1, ..., 2:] = ks, vs
    q2 = torch.zeros(3, 12, 80, dtype=torch.bfloat16, device=DEV)[:, 2:10, 8:72]
    q2.copy_(q)
    room, room_l = torch.full((3, 9, 70), 5.0, dtype=torch.bfloat16, device=DEV), torch.full((3, 20), 5.0, device=DEV)
    out, lse = room[:, 1:, 2:66], room_l[:, 4:12]
    got = fsa.flash_dense_attn_with_quantized_kvcache_func(q2, k2, v2, scales[0, ..., 1:2], scales[1, ..., 2:], out=out, lse=lse, return_lse=True)
    done()
    assert got[0] is out and got[1] is lse and torch.equal(out, want) and torch.equal(lse, want_lse)
    out.fill_(5.0), lse.fill_(5.0)
    assert (room == 5).all() and (room_l == 5).all()
    empty = fsa.flash_dense_attn_with_quantized_kvcache_func(q[:0], k[:0], v[:0], ks[:0], vs[:0], page_table=torch.zeros(0, 1, dtype=torch.int32, device=DEV),
                                                             skip_checks=True)
    assert empty.shape == (0, 8, 64)
    none = fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs, gather_kv_indices=torch.empty(3, 0, dtype=torch.int32, device=DEV), return_lse=True)
    done()
    assert not none[0].any() and (none[1] == -torch.inf).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pages that lie more than 2^32 bytes into the pool."""
    import flash_sparse_attn as fsa

    pages, page, hkv, d = 4200, 256, 32, 128  # 4.4 GB of codes
    small = make_cache(1, 3, page, hkv, d, "int8")
    big = torch.zeros(pages, hkv, page, d, dtype=torch.int8, device=DEV).transpose(1, 2)
    scales = torch.zeros(2, pages, hkv, page, 1, device=DEV)
    where = torch.tensor([[4199, 1, 4100]], dtype=torch.int32, device=DEV)
    at = where[0].long()
    big[at] = small[0]
    scales[0].transpose(1, 2)[at], scales[1].transpose(1, 2)[at] = small[2], small[3]
    q, used = normal(2, 1, 64, d), torch.tensor([700], dtype=torch.int32, device=DEV)
    flat = torch.arange(3, dtype=torch.int32, device=DEV)[None]
    want = fsa.flash_dense_attn_with_quantized_kvcache_func(q, small[0], small[0], small[2], small[3], page_table=flat, seqused_k=used)
    got = fsa.flash_dense_attn_with_quantized_kvcache_func(q, big, big, scales[0].transpose(1, 2), scales[1].transpose(1, 2), page_table=where, seqused_k=used)
    done()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_two_captured_calls_and_another_stream(kind):
    """Calls of two graphs replayed at a time on two streams, each with the workspace that was its own at capture."""
    import flash_sparse_attn as fsa

    sets = [(normal(i, 5, 8, 128),) + make_cache(10 + i, 5, 3000, 2, 128, kind) + (torch.tensor([3000, 1, 0, 77, 2000 + i], dtype=torch.int32, device=DEV),) for i in range(2)]
    want = [fsa.flash_dense_attn_with_quantized_kvcache_func(*s[:5], seqused_k=s[5]) for s in sets]
    done()
    graphs, kept, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s, st in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            kept.append(fsa.flash_dense_attn_with_quantized_kvcache_func(*s[:5], seqused_k=s[5]))
        graphs.append(g)
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    for st in streams:
        st.synchronize()
    done()
    for a, b in zip(kept, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 32)])
def test_a_serving_loop(kind, group):
    """A prompt with an image in it goes into the cache and through the forward operator on what was read back; then steps of one
    token: append, decode. Every result against attention over the values that the cache holds."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_quantized, empty_kv_quantized, read_kv_quantized

    b, hq, hkv, d, page, sections = 3, 8, 2, 128, 64, (16, 24, 24)
    cos, sin = tables(400, 64)
    cache = empty_kv_quantized(16, page, hkv, d, KINDS[kind], group_size=group)
    table = torch.full((b, 5), -1, dtype=torch.int32, device=DEV)
    free, count = torch.randperm(16, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(DEV), torch.tensor([16], dtype=torch.int32, device=DEV)
    used, lens = torch.zeros(b, dtype=torch.int32, device=DEV), [70, 1, 130]
    pool = dict(page_table=table, free_pages=free, free_count=count)
    cu = torch.tensor([0, 70, 71, 201], dtype=torch.int32, device=DEV)
    q, k, v = normal(1, 201, hq, d), normal(2, 201, hkv, d), normal(3, 201, hkv, d)
    place = torch.cat([torch.arange(n) for n in lens])
    ids = torch.stack([place // 16 * 16, place // 16, place % 16]).to(DEV)
    oq = append_kv_quantized(q, k, v, *cache, used, cos, sin, cu_seqlens_new=cu, position_ids=ids, sections=sections, **pool)
    rk, rv = read_kv_quantized(*cache, used, page_table=table, cu_seqlens=cu, total=201)
    out = fsa.flash_dense_attn_varlen_func(oq, rk, rv, cu, cu, 130, 130, is_causal=True)
    done()
    assert used.tolist() == lens
    for i in range(b):
        at = slice(int(cu[i]), int(cu[i + 1]))
        qq, kk, vv = oq[at].double(), rk[at].double().repeat_interleave(4, 1), rv[at].double().repeat_interleave(4, 1)
        s = torch.einsum("qhd,khd->hqk", qq, kk) * d**-0.5
        s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -torch.inf)
        want = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv)
        size = torch.einsum("hqk,khd->qhd", s.softmax(-1), vv.abs())
        # probabilities and the result are rounded to bf16: half a step each
        assert ((out[at].double() - want).abs() <= 2.0**-8 * 1.05 * (size + want.abs()) + 1e-4).all()
    for step in range(3):
        q, k, v = normal(10 + step, b, 1, hq, d), normal(20 + step, b, 1, hkv, d), normal(30 + step, b, 1, hkv, d)
        at = (used.long()[None, :, None] + 5).expand(3, b, 1)
        oq = append_kv_quantized(q, k, v, *cache, used, cos, sin, position_ids=at, sections=sections, **pool)
        out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(oq[:, 0], *cache, page_table=table, seqused_k=used, return_lse=True)
        done()
        all_k, all_v = values(cache[0], cache[2]), values(cache[1], cache[3])
        rows = [[x[table[i, :-(-n // page)].long().cpu()].flatten(0, 1)[:n] for i, n in enumerate(used.tolist())] for x in (all_k, all_v)]
        assert used.tolist() == [n + step + 1 for n in lens]
        reach = [3 * x.abs().amax((0, 1)) + x.abs().max() for x in (all_k, all_v)]  # above codes and centres taken apart
        check(out, lse, oq[:, 0], rows[0], rows[1], *reach)


def test_refusals_on_the_cpu():
    import flash_sparse_attn as fsa
    from flash_sparse_attn import _lib
    from flash_sparse_attn.ops.triton import flash_quant_dec
    from flash_sparse_attn.utils.kvcache import empty_kv_quantized

    i32 = torch.int32
    k, v, ks, vs = empty_kv_quantized(3, 64, 2, 64, device="cpu")
    q, table, used, at = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(3, 5, dtype=i32)
    good = dict(query=q, key=k, value=v, key_scales=ks, value_scales=vs, softmax_scale=None, page_table=None, gather_kv_indices=None, seqused_k=None, out=None, lse=None)
    flash_quant_dec._check(**good)
    flash_quant_dec._check(**dict(good, page_table=table, seqused_k=used, gather_kv_indices=at, out=q.clone(), lse=torch.zeros(3, 8)))
    odd = torch.zeros(3 * 8 * 64 + 1, dtype=torch.bfloat16)[1:].view(3, 8, 64)
    for bad in (dict(query=q[0]), dict(query=q.float()), dict(query=q[:, :7]), dict(query=q[:, :0]), dict(query=q[..., :32]), dict(query=q[:2]), dict(query=odd), dict(value=v[:, :32]),
                dict(key_scales=ks.half()), dict(page_table=table.long()), dict(page_table=table[:2]), dict(seqused_k=used[:2]), dict(seqused_k=used.long()),
                dict(gather_kv_indices=at.long()), dict(gather_kv_indices=at[:2]), dict(gather_kv_indices=at[0]), dict(gather_kv_indices=torch.zeros(3, 10, dtype=i32)[:, ::2]),
                dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(out=q[:2]), dict(out=q.half()), dict(out=odd),
                dict(out=q[:1].expand(3, 8, 64)), dict(lse=torch.zeros(3, 8).half()), dict(lse=torch.zeros(1, 8).expand(3, 8)),
                dict(page_table=table, key=k[:, :48], value=v[:, :48], key_scales=ks[:, :48], value_scales=vs[:, :48])):
        with pytest.raises(AssertionError):
            flash_quant_dec._check(**dict(good, **bad))
    with pytest.raises(RuntimeError, match="CUDA"):
        fsa.flash_dense_attn_with_quantized_kvcache_func(q, k, v, ks, vs)
    lib = _lib.load()

    def call(cache={}, **kw):
        a = _lib.FsaQuantDecodeArgs()
        for n in ("k", "v", "k_scales", "v_scales"):
            setattr(a.cache, n, 256)
        a.cache.heads_kv, a.cache.head_dim, a.cache.capacity = 1, 64, 8
        for n in ("q", "out", "lse", "ws", "status"):
            setattr(a, n, 256)
        a.batch, a.heads_q, a.dtype, a.softmax_scale = 1, 4, _lib.DT_BF16, 1.0
        for n, x in cache.items():
            setattr(a.cache, n, x)
        for n, x in kw.items():
            setattr(a, n, x)
        return lib.fsa_decode_quantized(ctypes.byref(a), None), lib.fsa_decode_quantized_workspace_bytes(ctypes.byref(a))

    pages = dict(page_table=256, page_size=32, max_pages=1, num_pages=1)
    for kw in (dict(q=None), dict(out=None), dict(lse=None), dict(ws=None), dict(status=None), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")),
               dict(softmax_scale=float("inf")), dict(q=264), dict(ws=264), dict(out=258), dict(q_stride_b=4), dict(o_stride_h=3)):
        rc, room = call(**kw)
        assert rc == -1 and room > 0, kw
    for kw in (dict(cache=dict(k=None)), dict(cache=dict(k=264)), dict(cache=dict(heads_kv=3)), dict(cache=dict(capacity=0)), dict(cache=dict(v_stride_b=8)), dict(batch=0),
               dict(heads_q=0), dict(topk=-1), dict(cache=dict(pages, max_pages=0))):
        assert call(**kw) == (-1, -1), kw
    for kw in (dict(cache=dict(format=5)), dict(cache=dict(head_dim=72)), dict(cache=dict(head_dim=256)), dict(cache=dict(format=2, group=48)),
               dict(cache=dict(pages, page_size=24)), dict(batch=1 << 30, heads_q=32, cache=dict(heads_kv=4))):
        assert call(**kw) == (-2, -2), kw
    assert call(dtype=_lib.DT_F32)[0] == -2
