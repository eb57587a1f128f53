"""Rows that are appended to a cache turned by their position: contiguous and paged caches, packed chunks, pages off the stack,
FP8, rows without room, against the definition in 64 bits; then the decode on what was stored; and refusals."""

import ctypes

import pytest
import torch

from test_rotary import check, done, launcher, normal, tables, turn  # noqa: F401

DEV = "cuda"
FP8_TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def check_fp8(got, want, size, scale):
    """Half a step of the format (relative 2^-4 or 2^-3; below its normal values half of the smallest step), of what saturates
    the largest value; 2^-22 of what is added up for the fp32 arithmetic, 2^-23 for the division."""
    info = torch.finfo(got.dtype)
    top = FP8_TOP[got.dtype]
    want = (want / scale).clamp(-top, top)
    bound = info.eps / 2 * want.abs() * (1 + 2.0**-10) + 2.0**-22 * size / scale + info.smallest_normal * info.eps / 2
    wrong = (got.float().double().cpu() - want).abs() > bound
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()} elements"


class Plain:
    """The append, row by row."""

    def __init__(self, kc, vc, used, table=None, free=None, count=0, pages=None):
        self.kc, self.vc, self.used = kc.double().cpu(), vc.double().cpu(), used.tolist()
        self.size = torch.zeros_like(self.kc)
        self.table = None if table is None else table.tolist()
        self.free, self.count = None if free is None else free.tolist(), count
        self.k_rows = torch.zeros(kc.shape[:2], dtype=torch.bool)
        self.stored = []

    def append(self, q, k, v, cos, sin, new, offset=0, interleaved=False):
        """q, k, v packed. Returns the turned queries; rows without room are zeros and end their sequence."""
        oq, oz, row = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
        offs = offset if isinstance(offset, list) else [offset] * len(new)
        for b, n in enumerate(new):
            reach = n
            cap = self.kc.shape[1] if self.table is None else len(self.table[b]) * self.kc.shape[1]
            reach = max(0, min(n, cap - self.used[b], cos.shape[0] - self.used[b] - offs[b]))
            if self.used[b] + offs[b] < 0:
                reach = 0
            kept = reach
            if self.table is not None and reach:
                page = self.kc.shape[1]
                for i in range(self.used[b] // page, (self.used[b] + reach - 1) // page + 1):
                    if self.table[b][i] < 0 and self.free is not None and self.count > 0:
                        self.count -= 1
                        self.table[b][i] = self.free[self.count]
                    if not 0 <= self.table[b][i] < self.kc.shape[0]:
                        kept = min(kept, max(0, i * page - self.used[b]))
            self.stored.append(kept)
            for t in range(kept):
                slot = self.used[b] + t
                at = (self.table[b][slot // self.kc.shape[1]], slot % self.kc.shape[1]) if self.table is not None else (b, slot)
                c, s = cos[slot + offs[b]], sin[slot + offs[b]]
                oq[row + t], oz[row + t] = turn(q[row + t], c, s, interleaved)
                self.kc[at], self.size[at] = turn(k[row + t], c, s, interleaved)
                self.vc[at] = v[row + t].double().cpu()
                self.k_rows[at] = True
            row += n
        return oq, oz


def pages_for(gen, used, slots, page, spare=2):
    """A table that holds the pages of `used` positions, scattered, and the stack of the others."""
    pool = len(used) * slots + spare
    perm = torch.randperm(pool, generator=gen).tolist()
    table = torch.full((len(used), slots), -1, dtype=torch.int32)
    for b, u in enumerate(used):
        for i in range(-(-u // page)):
            table[b, i] = perm.pop()
    free = torch.tensor(perm + [0] * (pool - len(perm)), dtype=torch.int32)
    return pool, table, free, len(perm)


def run(case):
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    g = torch.Generator().manual_seed(case.get("seed", 0))
    dt, cdt = case.get("dtype", torch.bfloat16), case.get("cache", None)
    cdt = cdt or dt
    new, used = case["new"], case["used"]
    b, total, hq, hkv, d = len(new), sum(new) + case.get("behind", 0), case.get("hq", 4), case.get("hkv", 2), case.get("d", 64)
    packed = case.get("packed", False)
    half, il = case.get("half", d // 2), case.get("interleaved", False)
    offset = case.get("offset", 0)
    cos, sin = tables(case.get("rows", 600), half)
    q, k, v = normal(1, total, hq, d, dtype=dt), normal(2, total, hkv, d, dtype=dt), normal(3, total, hkv, d, dtype=dt)
    page = case.get("page", 0)
    table = free = count = None
    if page:
        pool, table, free, height = pages_for(g, used, case["slots"], page)
        height = case.get("height", height)
        if "break_table" in case:
            table[case["break_table"]] = case.get("bad_page", pool)
        if not case.get("stack", True):
            free = None
        shape = (pool, page, hkv, d)
    else:
        shape = (b, case["capacity"], hkv, d)
    kc, vc = (normal(4 + i, *shape, dtype=dt).to(cdt) for i in range(2))
    before = kc.clone(), vc.clone()
    plain = Plain(kc, vc, torch.tensor(used), table, free, height if page else 0)
    oq, oz = plain.append(q[:sum(new)], k, v, cos, sin, new, offset, il)
    used_d = torch.tensor(used, dtype=torch.int32, device=DEV)
    kw = {}
    if page:
        table = table.to(DEV)
        kw["page_table"] = table
        if free is not None:
            count = torch.tensor([height], dtype=torch.int32, device=DEV)
            kw.update(free_pages=free.to(DEV), free_count=count)
    if offset:
        kw["seqlen_offsets"] = offset if isinstance(offset, int) else torch.tensor(offset, dtype=torch.int32, device=DEV)
    scales = (1.0, 1.0, 1.0)
    if cdt in FP8_TOP:
        scales = case.get("scales", (0.03, 0.011, 0.007))
        kw.update({n: torch.tensor([s], device=DEV) for n, s in zip(("query_scale", "key_scale", "value_scale"), scales)})
        scales = [float(torch.tensor(s)) for s in scales]
    shape = (lambda t: t) if packed else (lambda t: t.view(b, -1, *t.shape[1:]))
    if packed:
        kw["cu_seqlens_new"] = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    advance = case.get("advance", True)
    query = None if case.get("no_query") else shape(q)
    got = append_kv_rotary(query, shape(k), shape(v), kc, vc, used_d, cos, sin, interleaved=il, advance=advance, **kw)
    torch.cuda.synchronize()
    assert used_d.tolist() == [u + (s if advance else 0) for u, s in zip(used, plain.stored)]
    if page:
        assert table.tolist() == plain.table
        if count is not None:
            assert int(count) == plain.count
    rows = plain.k_rows.to(DEV)
    for cache, old in ((kc, before[0]), (vc, before[1])):
        assert torch.equal(cache[~rows].float(), old[~rows].float())  # what no row was meant for
    if cdt in FP8_TOP:
        check_fp8(kc[rows], plain.kc[rows.cpu()], plain.size[rows.cpu()], scales[1])
        check_fp8(vc[rows], plain.vc[rows.cpu()], torch.zeros_like(plain.vc[rows.cpu()]), scales[2])
    else:
        check(kc[rows], plain.kc[rows.cpu()], plain.size[rows.cpu()])
        assert torch.equal(vc[rows].double().cpu(), plain.vc[rows.cpu()])
    if case.get("no_query"):
        assert got is None
    else:
        flat = got.reshape(-1, hq, d)
        assert flat.dtype == cdt and not flat[sum(new):].float().any()
        if cdt in FP8_TOP:
            check_fp8(flat[:sum(new)], oq, oz, scales[0])
        else:
            check(flat[:sum(new)], oq, oz)
    return plain, new


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(new=[1], used=[0], capacity=1),
    dict(new=[1], used=[37], capacity=100, dtype=torch.float16, interleaved=True),
    dict(new=[1] * 9, used=[0, 1, 5, 63, 64, 65, 99, 98, 3], capacity=100, d=128, hq=16, hkv=2),
    dict(new=[3] * 4, used=[0, 10, 90, 97], capacity=100, offset=400),
    dict(new=[3] * 4, used=[0, 10, 90, 97], capacity=100, offset=[0, 5, 500, 33], advance=False),
    dict(new=[0, 7, 1, 0, 130], used=[4, 0, 9, 0, 20], capacity=150, packed=True, behind=5),
    dict(new=[0, 0], used=[4, 0], capacity=150, packed=True, behind=3),
    dict(new=[200] * 3, used=[1, 0, 7], capacity=300, d=96, half=24, no_query=True),
    dict(new=[300] * 8, used=[3] * 8, capacity=303, d=128, hq=8, hkv=8),
    dict(new=[5] * 3, used=[0, 1, 2], capacity=10, d=48, half=10, hq=6, hkv=3),
    dict(new=[5] * 3, used=[0, 1, 2], capacity=10, d=80, half=20, interleaved=True, hq=5, hkv=1),
], ids=lambda c: f"{len(c['new'])}x{max(c['new'])}")
def test_contiguous_caches(case):
    run(case)
    done()


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("case", [
    dict(new=[1] * 5, used=[0, 31, 32, 33, 64], page=32, slots=4),
    dict(new=[1] * 5, used=[0, 30, 32, 33, 95], page=32, slots=3, d=128, hq=32, hkv=4),
    dict(new=[40] * 3, used=[0, 31, 60], page=32, slots=4, offset=17),
    dict(new=[0, 64, 100, 1, 0, 33], used=[5, 64, 0, 63, 0, 30], page=64, slots=3, packed=True, behind=2),
    dict(new=[500, 3], used=[11, 0], page=32, slots=16, packed=True, rows=700),
    dict(new=[1] * 1100, used=[i % 70 for i in range(1100)], page=64, slots=2, hq=1, hkv=1, d=32),
    dict(new=[130] * 40, used=[i % 70 for i in range(40)], page=32, slots=7, hq=1, hkv=1, d=32),
], ids=lambda c: f"{len(c['new'])}x{max(c['new'])}p{c['page']}")
def test_paged_caches_with_pages_off_the_stack(case, cache):
    run(dict(case, cache=cache))
    done()


@pytest.mark.gpu
def test_saturation_and_special_values_in_fp8():
    run(dict(new=[4] * 3, used=[0, 1, 2], capacity=10, cache=torch.float8_e4m3fn, scales=(0.001, 0.002, 0.004)))
    run(dict(new=[4] * 3, used=[0, 1, 2], capacity=10, cache=torch.float8_e5m2, scales=(1e-5, 2e-6, 1e-5)))
    done()
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    cos, sin = tables(4, 8)
    kc, one = torch.zeros(1, 4, 1, 16, device=DEV).to(torch.float8_e4m3fn), torch.ones(1, device=DEV)
    vc, used = kc.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.ones(1, 1, 1, 16, dtype=torch.bfloat16, device=DEV)
    x[..., 3], x[..., 5] = float("nan"), float("-inf")
    append_kv_rotary(None, torch.ones_like(x), x, kc, vc, used, cos, sin, key_scale=one, value_scale=one)
    row = vc[0, 0, 0].float()
    assert torch.isnan(row[3]) and row[5] == -448 and row[0] == 1 and torch.isfinite(row).sum() == 15


@pytest.mark.gpu
@pytest.mark.parametrize("status,case", [
    (3, dict(new=[3] * 4, used=[0, 8, 9, 12], capacity=10)),                                      # ends inside, and behind the end
    (3, dict(new=[40] * 3, used=[0, 31, 60], page=32, slots=3)),                                  # the table ends
    (3, dict(new=[40] * 4, used=[0, 31, 60, 5], page=32, slots=4, height=2)),                     # the stack does
    (3, dict(new=[1] * 4, used=[0, 32, 60, 64], page=32, slots=4, height=0)),
    (3, dict(new=[40] * 3, used=[0, 31, 60], page=32, slots=4, stack=False)),                     # nobody assigned them
    (3, dict(new=[40] * 3, used=[0, 31, 60], page=32, slots=4, break_table=(1, 1))),              # a page that does not exist
    (3, dict(new=[1] * 3, used=[0, 31, 60], page=32, slots=4, break_table=(2, 1), bad_page=1 << 30)),
    (5, dict(new=[3] * 4, used=[0, 8, 9, 5], capacity=12, rows=9)),
    (5, dict(new=[3] * 4, used=[0, 8, 9, 5], capacity=12, offset=[-1, -8, -20, 0])),
    (3, dict(new=[40, 0, 9], used=[0, 31, 3], page=32, slots=4, packed=True, height=1)),
], ids=str)
def test_rows_without_room_end_their_sequence_and_are_reported(status, case):
    import flash_sparse_attn as fsa

    plain, new = run(case)
    assert plain.stored != list(new)
    with pytest.raises(RuntimeError, match=f"device status {status}"):
        fsa.check_status()


@pytest.mark.gpu
def test_rows_far_into_a_large_cache():
    """Offsets that pass 32 bits: 2.2e9 elements in front of the row."""
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    pages, page, h, d = 17000, 256, 4, 128
    pool = torch.zeros(pages, page, h, d, dtype=torch.bfloat16, device=DEV)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    used = torch.tensor([255], dtype=torch.int32, device=DEV)
    cos, sin = tables(300, 64)
    k = normal(1, 1, 1, h, d)
    append_kv_rotary(None, k, k, pool, pool.clone(), used, cos, sin, page_table=table)
    done()
    check(pool[-1, 255][None], *turn(k[0], cos[255:256], sin[255:256], False))
    pool[-1, 255] = 0
    assert not pool.any()


@pytest.mark.gpu
def test_tokens_outside_every_sequence():
    """Packed bounds that begin behind the first token and end behind the last: nothing is stored that is not there."""
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    cos, sin = tables(40, 16)
    q, k, v = normal(1, 9, 2, 32), normal(2, 9, 1, 32), normal(3, 9, 1, 32)
    kc = torch.zeros(3, 20, 1, 32, dtype=torch.bfloat16, device=DEV)
    vc, used = torch.zeros_like(kc), torch.tensor([0, 5, 19], dtype=torch.int32, device=DEV)
    cu = torch.tensor([2, 4, 4, 30], dtype=torch.int32, device=DEV)
    out = append_kv_rotary(q, k, v, kc, vc, used, cos, sin, cu_seqlens_new=cu)
    torch.cuda.synchronize()
    assert used.tolist() == [2, 5, 20]  # two rows, none, and the one of five that there is room for
    assert not out[:2].any() and not out[5:].any() and torch.equal(vc[0, :2], v[2:4]) and torch.equal(vc[2, 19], v[4])
    assert not vc[0, 2:].any() and not vc[1].any() and not vc[2, :19].any()
    check(out[2:4], *turn(q[2:4], cos[:2], sin[:2], False))
    check(out[4:5], *turn(q[4:5], cos[19:20], sin[19:20], False))
    import flash_sparse_attn as fsa

    with pytest.raises(RuntimeError, match="device status 3"):
        fsa.check_status()


@pytest.mark.gpu
def test_strided_rows_and_result_buffer():
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    b, hq, hkv, d = 3, 4, 2, 64
    cos, sin = tables(64, 32)
    fused = normal(1, b, 1, (hq + 2 * hkv) * d)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in fused.split((hq * d, hkv * d, hkv * d), -1))
    caches = torch.zeros(2, b, hkv, 40, d, dtype=torch.bfloat16, device=DEV)  # heads in front of positions, one buffer
    kc, vc = caches[0].transpose(1, 2), caches[1].transpose(1, 2)
    used = torch.tensor([0, 20, 39], dtype=torch.int32, device=DEV)
    buf = torch.zeros(b, 1, hq, 2 * d, dtype=torch.bfloat16, device=DEV)
    out = append_kv_rotary(q, k, v, kc, vc, used, cos, sin, out=buf[..., :d])
    done()
    at = torch.tensor([0, 20, 39])
    assert out.data_ptr() == buf.data_ptr() and not buf[..., d:].any()
    check(buf[:, 0, :, :d], *turn(q[:, 0], cos.cpu()[at], sin.cpu()[at], False))
    check(kc[torch.arange(b), at], *turn(k[:, 0], cos.cpu()[at], sin.cpu()[at], False))
    assert torch.equal(vc[torch.arange(b), at], v[:, 0]) and used.tolist() == [1, 21, 40]


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float8_e4m3fn])
def test_steps_in_a_replayed_graph_feed_the_decode(cache):
    """A serving loop: prompts, then captured steps of one token (append, decode), pages taken on the way."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    b, hq, hkv, d, page, slots = 3, 8, 2, 128, 32, 4
    pool = b * slots
    kc = torch.zeros(pool, page, hkv, d, dtype=torch.bfloat16, device=DEV).to(cache)
    vc = kc.clone()
    table = torch.full((b, slots), -1, dtype=torch.int32, device=DEV)
    free, count = torch.arange(pool, dtype=torch.int32, device=DEV), torch.tensor([pool], dtype=torch.int32, device=DEV)
    used = torch.zeros(b, dtype=torch.int32, device=DEV)
    cos, sin = tables(slots * page, d // 2)
    fp8 = cache != torch.bfloat16
    scale = torch.full((1,), 2.0**-6, device=DEV)
    scales = dict(query_scale=scale, key_scale=scale, value_scale=scale) if fp8 else {}
    kw = dict(page_table=table, free_pages=free, free_count=count, **scales)
    prompts = [30, 1, 64]
    rows = normal(1, 3, sum(prompts) + 40 * b, hkv, d)
    queries = normal(2, 40, b, 1, hq, d)
    cu = torch.tensor([0, 30, 31, 95], dtype=torch.int32, device=DEV)
    append_kv_rotary(None, rows[0, :95], rows[1, :95], kc, vc, used, cos, sin, cu_seqlens_new=cu, **kw)
    q, k, v = queries[0].clone(), rows[0, 95:95 + b, None].clone(), rows[1, 95:95 + b, None].clone()

    def step():
        turned = append_kv_rotary(q, k, v, kc, vc, used, cos, sin, **kw)
        return fsa.flash_dense_attn_with_kvcache_func(turned[:, 0], kc, vc, page_table=table, seqused_k=used, is_quant=fp8, **scales)

    state = [t.clone() for t in (used, table, count)]
    step()  # warm; its row is written again below
    for t, old in zip((used, table, count), state):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    keys = [[rows[0, a:e].cpu()] for a, e in ((0, 30), (30, 31), (31, 95))]
    values = [[rows[1, a:e].cpu()] for a, e in ((0, 30), (30, 31), (31, 95))]
    for i in range(40):
        at = 95 + i * b
        q.copy_(queries[i]), k.copy_(rows[0, at:at + b, None]), v.copy_(rows[1, at:at + b, None])
        graph.replay()
        for s in range(b):
            keys[s].append(rows[0, at + s:at + s + 1].cpu())
            values[s].append(rows[1, at + s:at + s + 1].cpu())
        if i not in (0, 1, 33, 39):
            continue
        for s in range(b):
            ks, vs = torch.cat(keys[s]), torch.cat(values[s]).double()
            n = ks.shape[0]
            kt, qt = turn(ks, cos[:n], sin[:n], False)[0], turn(queries[i, s], cos[n - 1:n], sin[n - 1:n], False)[0][0]
            score = torch.einsum("gqd,ngd->gqn", qt.view(hkv, hq // hkv, d), kt) / d**0.5
            want = torch.einsum("gqn,ngd->gqd", score.softmax(-1), vs).reshape(hq, d)
            # bf16: results and values below 4, half a step of the result 2^-8 * 2 = 0.008, of keys, queries and probabilities as
            # much again in all. e4m3: values below 4 are off by up to 0.125; scores by 0.04 in the root mean square (128 products of
            # two factors with 0.026 each, over sqrt(128)), four times that by chance, probabilities by up to a quarter of it,
            # times differences of values below 3.
            assert (out[s].double().cpu() - want).abs().max() < (0.25 if fp8 else 2e-2)
    done()
    assert used.tolist() == [70, 41, 104] and int(count) == pool - (3 + 2 + 4)


def test_refusals():
    from flash_sparse_attn import _lib
    from flash_sparse_attn.utils import kvcache

    b, t, hq, hkv, d = 2, 3, 4, 2, 64
    bf, i32 = torch.bfloat16, torch.int32
    cos, sin = tables(50, 32, device="cpu")
    good = dict(query=torch.zeros(b, t, hq, d, dtype=bf), key_new=torch.zeros(b, t, hkv, d, dtype=bf),
                value_new=torch.zeros(b, t, hkv, d, dtype=bf), key_cache=torch.zeros(b, 9, hkv, d, dtype=bf),
                value_cache=torch.zeros(b, 9, hkv, d, dtype=bf), seqused_k=torch.zeros(b, dtype=i32), cos=cos, sin=sin, page_table=None,
                free_pages=None, free_count=None, cu_seqlens_new=None, query_scale=None, key_scale=None, value_scale=None, out=None)
    table, one = torch.zeros(b, 2, dtype=i32), torch.ones(1)
    kvcache._check_append(**good)
    kvcache._check_append(**dict(good, page_table=table, free_pages=table[0], free_count=torch.zeros(1, dtype=i32)))
    f8 = good["key_cache"].to(torch.float8_e4m3fn)
    kvcache._check_append(**dict(good, key_cache=f8, value_cache=f8, query_scale=one, key_scale=one, value_scale=one))
    for bad in (dict(query=good["query"].half()), dict(query=good["query"][:, :2]), dict(query=good["query"][:, :, :3]),
                dict(value_new=good["value_new"][:, :2]), dict(key_new=good["key_new"].float(), value_new=good["value_new"].float()),
                dict(key_cache=good["key_cache"][:1], value_cache=good["value_cache"][:1]), dict(value_cache=good["value_cache"][:, :8]),
                dict(key_cache=good["key_cache"].half(), value_cache=good["value_cache"].half()), dict(key_cache=f8, value_cache=f8),
                dict(key_scale=one), dict(seqused_k=torch.zeros(b)), dict(seqused_k=torch.zeros(3, dtype=i32)), dict(page_table=table[:1]),
                dict(page_table=table.long()), dict(free_pages=table[0]), dict(page_table=table, free_pages=table[0]),
                dict(cu_seqlens_new=torch.zeros(3, dtype=i32)), dict(cos=cos[:, :16]), dict(out=good["query"][:, :2]),
                dict(out=good["query"].half()), dict(query=None, out=good["query"]), dict(key_new=good["key_new"].transpose(2, 3).contiguous().transpose(2, 3)),
                dict(key_cache=good["key_cache"][:, :1].expand(b, 9, hkv, d)), dict(value_cache=good["value_cache"][:1].expand(b, 9, hkv, d)),
                dict(out=good["query"][:1].expand(b, t, hq, d)), dict(page_table=table[:1].expand(b, 2)),
                dict(page_table=torch.zeros(2, b, dtype=i32).T[:, :2] if b != 2 else torch.zeros(b, 4, dtype=i32)[:, ::2])):
        with pytest.raises(AssertionError):
            kvcache._check_append(**dict(good, **bad))
    args = {n: good[n] for n in ("query", "key_new", "value_new", "key_cache", "value_cache", "seqused_k", "cos", "sin")}
    with pytest.raises(RuntimeError, match="CUDA"):
        kvcache.append_kv_rotary(**args)
    lib = _lib.load()

    def call(**kw):
        a = _lib.FsaKvAppendRotaryArgs()
        a.k_new = a.v_new = a.k_cache = a.v_cache = a.cos = a.sin = a.seqused_k = a.place_ws = a.status = 256
        a.batch, a.new_tokens, a.heads_kv, a.head_dim, a.rotary_dim, a.table_rows, a.capacity = 1, 1, 1, 64, 64, 1, 1
        a.dtype = a.cache_dtype = _lib.DT_BF16
        a.table_dtype = _lib.DT_F32
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.fsa_kv_append_rotary(ctypes.byref(a), None)

    for kw in (dict(k_new=None), dict(v_cache=None), dict(place_ws=None, free_pages=256, free_count=256, page_table=256, page_size=32, max_pages=1, num_pages=1), dict(heads_q=4), dict(k_new=257), dict(k_cache=257), dict(capacity=0),
               dict(page_table=256, page_size=0, max_pages=1, num_pages=1), dict(page_table=256, page_size=32, max_pages=0, num_pages=1),
               dict(page_table=256, page_size=32, max_pages=1, num_pages=0), dict(free_pages=256, free_count=256),
               dict(page_table=256, page_size=32, max_pages=1, num_pages=1, free_pages=256), dict(cache_dtype=_lib.DT_E4M3),
               dict(rotary_dim=128), dict(new_tokens=-1)):
        assert call(**kw) == -1, kw
    assert call(cache_dtype=_lib.DT_FP16) == -2 and call(dtype=_lib.DT_F32) == -2 and call(new_tokens=0) == 0


def test_argument_blocks_match_the_header():
    import os
    import re

    from flash_sparse_attn import _lib

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fsa_b200.h")).read()
    for name in ("FsaRotaryArgs", "FsaKvAppendRotaryArgs"):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1), flags=re.S)
        fields = [re.findall(r"[A-Za-z_]\w*", part)[-1] for stmt in body.split(";") if stmt.strip() for part in stmt.split(",")]
        assert fields == [f[0] for f in getattr(_lib, name)._fields_]


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [False, True])
def test_a_gradient_notices_lengths_that_were_advanced(rotary):
    """A rotation keeps its offsets for the gradient: when an append has advanced them in place that gradient would be another one's.
    Autograd has to say so. Lengths that stay may be used."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv, append_kv_rotary

    cos, sin = tables(20, 16)
    x, k = normal(1, 2, 1, 2, 32).requires_grad_(), normal(2, 2, 1, 2, 32)
    kc = torch.zeros(2, 9, 2, 32, dtype=torch.bfloat16, device=DEV)
    vc, used = torch.zeros_like(kc), torch.tensor([3, 5], dtype=torch.int32, device=DEV)
    want = turn(torch.ones_like(k), cos[used.long()][:, None], sin[used.long()][:, None], False, -1)
    y = fsa.apply_rotary_func(x, None, cos, sin, seqlen_offsets=used)
    append_kv_rotary(None, k, k, kc, vc, used, cos, sin, advance=False)
    (d,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    check(d, *want)
    if rotary:
        append_kv_rotary(None, k, k, kc, vc, used, cos, sin)
    else:
        append_kv(k, k, kc, vc, used)
    done()
    assert used.tolist() == [4, 6]
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.inference_mode():  # lengths that autograd does not follow at all
        more = torch.tensor([3, 5], dtype=torch.int32, device=DEV)
    (append_kv_rotary(None, k, k, kc, vc, more, cos, sin) if rotary else append_kv(k, k, kc, vc, more))
    done()
    assert more.tolist() == [4, 6]


@pytest.mark.gpu
def test_a_gradient_notices_a_result_buffer_that_was_written():
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    cos, sin = tables(20, 16)
    q, k = normal(1, 1, 1, 2, 32), normal(2, 1, 1, 1, 32)
    kc = torch.zeros(1, 9, 1, 32, dtype=torch.bfloat16, device=DEV)
    vc, used, out = torch.zeros_like(kc), torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones_like(q)
    w = torch.ones_like(q).requires_grad_()
    y = (w * out).sum()
    append_kv_rotary(q, k, k, kc, vc, used, cos, sin, out=out)
    done()
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("form", [dict(d=128, half=32), dict(d=40, half=10, interleaved=True)], ids=["128", "40"])
def test_many_rows_in_packed_chunks(form, cache):
    """Enough elements for threads that take several heads of a row each, of 6 query, 2 key and 2 value heads; pages off the stack."""
    run(dict(form, new=[1300, 0, 1, 1700, 900], used=[5, 9, 63, 64, 0], page=64, slots=28, packed=True, behind=2, hq=6, hkv=2, rows=1800, cache=cache))
    done()
