"""Operators measured against their plain forms: rotary positions with their gradient, the append of rotated rows to a
cache, and decode attention over a prefix that the whole batch shares.

``own`` false: elementary torch operations in 32 bits, rounded once at the end. ``own`` true: the calls that a user
makes of the framework."""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-sparse-attention_b200")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"bf16": 2, "fp16": 2}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}


def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import flash_sparse_attn
    from flash_sparse_attn.utils import kvcache

    return flash_sparse_attn, kvcache


# ----------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # a training step of a decoder layer: batch of whole sequences, forward and gradient
        dict(name="rotary-train", op="rotary", packed=False, batch=4, seq=4096, lens=0, heads_q=32, heads_kv=8,
             head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16"),
        # packed training tokens of unequal sequences, half of each head's columns rotated in neighbouring pairs
        dict(name="rotary-packed", op="rotary", packed=True, batch=13, seq=2500, lens=11, heads_q=16, heads_kv=4,
             head_dim=64, rotary_dim=32, interleaved=True, dtype="fp16"),
        # one short sequence with an odd length, where the launch is what counts
        dict(name="rotary-short", op="rotary", packed=False, batch=1, seq=77, lens=0, heads_q=8, heads_kv=2,
             head_dim=96, rotary_dim=96, interleaved=False, dtype="bf16"),
        # a decode step of a serving batch: one token each, paged cache, pages assigned by the scheduler
        dict(name="append-step", op="append", packed=False, batch=64, new=1, lens=3, max_len=767, page=256, alloc=False,
             heads_q=64, heads_kv=8, head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", cache="bf16"),
        # prompt chunks of unequal length, pages taken from the stack of free ones on the way
        dict(name="append-chunks", op="append", packed=True, batch=16, new=4000, lens=5, max_len=1500, page=64, alloc=True,
             heads_q=32, heads_kv=8, head_dim=128, rotary_dim=128, interleaved=False, dtype="bf16", cache="bf16"),
        # four drafted tokens of each sequence into an FP8 cache
        dict(name="append-fp8", op="append", packed=False, batch=48, new=4, lens=7, max_len=91, page=32, alloc=False,
             heads_q=32, heads_kv=4, head_dim=128, rotary_dim=64, interleaved=False, dtype="bf16", cache="e4m3"),
        # one token of one user, contiguous cache
        dict(name="append-one", op="append", packed=False, batch=1, new=1, lens=2, max_len=2001, page=0, alloc=False,
             heads_q=16, heads_kv=4, head_dim=64, rotary_dim=64, interleaved=True, dtype="fp16", cache="fp16"),
        # a handful of samples from one short prompt: latency
        dict(name="prefix-few", op="prefix", batch=4, prefix=1000, lens=1, max_len=40, page=0, heads_q=8, heads_kv=2,
             head_dim=64, dtype="bf16"),
        # a chat service: system prompt of 8192 tokens, own turns of up to a thousand, pages of 64
        dict(name="prefix-chat", op="prefix", batch=64, prefix=8192, lens=4, max_len=1024, page=64, heads_q=32,
             heads_kv=8, head_dim=128, dtype="bf16"),
        # many samples of one long document: matrix products bound it
        dict(name="prefix-fanout", op="prefix", batch=256, prefix=32768, lens=6, max_len=256, page=256, heads_q=32,
             heads_kv=8, head_dim=128, dtype="bf16"),
        # a few questions about a very long document: the prefix's bytes bound it
        dict(name="prefix-long", op="prefix", batch=6, prefix=131072, lens=8, max_len=300, page=128, heads_q=64,
             heads_kv=8, head_dim=128, dtype="fp16"),
        # odd everything: five query heads per KV head, head size 96, lengths that end inside a tile
        dict(name="prefix-odd", op="prefix", batch=37, prefix=5001, lens=9, max_len=333, page=32, heads_q=20,
             heads_kv=4, head_dim=96, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "prefix"])
    dtype = rng.choice(["bf16", "fp16"])
    lens = rng.randrange(1, 1 << 30)
    heads_kv = rng.choice([1, 2, 3, 4, 8])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    head_dim = rng.choice([32, 48, 64, 80, 96, 112, 128])
    rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
    interleaved = rng.random() < 0.4
    if op == "rotary":
        packed = rng.random() < 0.5
        batch = _log_int(rng, 1, 32)
        seq = max(1, min(_log_int(rng, 1, 20000), 80_000_000 // (batch * (heads_q + heads_kv) * head_dim)))
        return dict(op=op, packed=packed, batch=batch, seq=seq, lens=lens, heads_q=heads_q, heads_kv=heads_kv,
                    head_dim=head_dim, rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype)
    if op == "append":
        packed = rng.random() < 0.5
        batch = _log_int(rng, 1, 128)
        new = rng.choice([1, 1, rng.randint(2, 8), max(1, min(_log_int(rng, 9, 4000), 32000 // batch))])
        page = rng.choice([0, 32, 64, 128, 256])
        cache = rng.choice([dtype, dtype, "e4m3", "e5m2"])
        max_len = _log_int(rng, 1, 2000 if cache == dtype else 100)
        return dict(op=op, packed=packed, batch=batch, new=new, lens=lens, max_len=max_len, page=page,
                    alloc=page > 0 and rng.random() < 0.5, heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim,
                    rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype, cache=cache)
    batch = _log_int(rng, 1, 300)
    prefix = max(1, min(_log_int(rng, 1, 131072), 250_000_000 // (batch * heads_q)))
    max_len = max(1, min(_log_int(rng, 1, 4000), 250_000_000 // (batch * heads_q), 60_000_000 // (batch * heads_kv * head_dim)))
    return dict(op=op, batch=batch, prefix=prefix, lens=lens, max_len=max_len, page=rng.choice([0, 32, 64, 128, 256]),
                heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim, dtype=dtype)


def _lengths(case, count, low, high, salt=0):
    """Unequal lengths that belong to the case (not to the seed): the first is the largest, one is the smallest."""
    rng = random.Random(case["lens"] * 7919 + salt)
    out = [high] + [rng.randint(low, high) for _ in range(count - 1)]
    if count > 2:
        out[rng.randrange(1, count)] = low
    return out


def _new_lengths(case):
    return _lengths(case, case["batch"], min(1, case["new"]), case["new"], 1) if case["packed"] else [case["new"]] * case["batch"]


def work(case):
    es, d = _BYTES[case["dtype"]], case["head_dim"]
    if case["op"] == "rotary":
        lens = _lengths(case, case["batch"], 1, case["seq"]) if case["packed"] else [case["seq"]] * case["batch"]
        elems = sum(lens) * (case["heads_q"] + case["heads_kv"]) * d
        table = 2 * 4 * max(lens) * case["rotary_dim"] // 2
        # forward and gradient: each reads and writes every element once
        return {"bytes": 4 * elems * es + 2 * table, "flops": 2 * 3 * elems * case["rotary_dim"] // d}
    if case["op"] == "append":
        tokens = sum(_new_lengths(case))
        cs = _BYTES.get(case["cache"], 1)
        qs = es if case["cache"] in _BYTES else 1
        q, kv = tokens * case["heads_q"] * d, tokens * case["heads_kv"] * d
        return {"bytes": q * (es + qs) + 2 * kv * (es + cs) + tokens * 4 * case["rotary_dim"],
                "flops": 3 * (q + kv) * case["rotary_dim"] // d}
    own_keys = sum(_lengths(case, case["batch"], 0, case["max_len"]))
    rows = case["batch"] * case["heads_q"]
    return {"bytes": (case["prefix"] + own_keys) * case["heads_kv"] * d * 2 * es + 2 * rows * d * es + 4 * rows,
            "flops": 4 * d * case["heads_q"] * (case["batch"] * case["prefix"] + own_keys)}


# ----------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------
def _tables(positions, rotary_dim):
    """cos and sin of position * 10000^(-2i / R): angles in 64 bits, kept in 32."""
    freq = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cuda") / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _pages(gen, batch, slots, pool):
    """A page table whose pages lie scattered over the pool."""
    perm = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    return perm[: batch * slots].view(batch, slots).contiguous(), perm


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _int32(out)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]

    def normal(*shape, dt=dtype):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    st = {"case": case}
    if case["op"] == "rotary":
        if case["packed"]:
            lens = _lengths(case, case["batch"], 1, case["seq"])
            st["cu"] = _cumulative(lens)
            lead = (sum(lens),)
        else:
            lead = (case["batch"], case["seq"])
        st["cos"], st["sin"] = _tables(case["seq"], case["rotary_dim"])
        st["q"], st["k"] = normal(*lead, hq, d).requires_grad_(), normal(*lead, hkv, d).requires_grad_()
        st["gq"], st["gk"] = normal(*lead, hq, d), normal(*lead, hkv, d)
        return st
    if case["op"] == "append":
        b, new = case["batch"], _new_lengths(case)
        used = _lengths(case, b, 0, case["max_len"], 2)
        lead = (sum(new),) if case["packed"] else (b, case["new"])
        st["cu"] = _cumulative(new) if case["packed"] else None
        st["q"], st["k"], st["v"] = normal(*lead, hq, d), normal(*lead, hkv, d), normal(*lead, hkv, d)
        capacity = case["max_len"] + case["new"]
        # the sequences continue a prompt of 50 tokens that lies elsewhere
        st["offset"] = 50
        st["cos"], st["sin"] = _tables(capacity + 50, case["rotary_dim"])
        st["used"] = _int32(used)
        fp8 = case["cache"] in _FP8
        # scales of q, k and v as a calibration leaves them: powers of two
        st["scales"] = [torch.tensor([s], dtype=torch.float32, device="cuda") for s in (2.0**-5, 2.0**-6, 2.0**-6)] if fp8 else None
        cache_dtype = _FP8[case["cache"]] if fp8 else dtype
        if case["page"]:
            slots = -(-capacity // case["page"])
            pool = b * slots + 3
            shape = (pool, case["page"], hkv, d)
            table, perm = _pages(gen, b, slots, pool)
            st["table"], st["free"], st["count"] = table, None, None
            if case["alloc"]:
                # only the pages that hold something are assigned; the rest is on the stack
                st["free"] = perm.flip(0).contiguous()
                held = (st["used"].long() + case["page"] - 1) // case["page"]
                st["table"] = torch.where(torch.arange(slots, device="cuda")[None, :] < held[:, None], table, -1).to(torch.int32)
                flags = torch.zeros(pool, dtype=torch.bool, device="cuda")
                flags[st["table"][st["table"] >= 0].long()] = True
                order = torch.argsort(flags[st["free"].long()].int(), stable=True)
                st["free"] = st["free"][order].contiguous()
                st["count"] = (pool - flags.sum()).to(torch.int32).reshape(1)
        else:
            shape = (b, capacity, hkv, d)
            st["table"] = st["free"] = st["count"] = None
        st["kc"], st["vc"] = normal(*shape).to(cache_dtype), normal(*shape).to(cache_dtype)
        return st
    b = case["batch"]
    lens = _lengths(case, b, 0, case["max_len"])
    st["q"], st["used"] = normal(b, hq, d), _int32(lens)
    if case["page"]:
        page = case["page"]
        slots, common = -(-case["max_len"] // page), -(-case["prefix"] // page)
        pool = b * slots + common
        table, perm = _pages(gen, b, slots, pool)
        st["table"], st["common"] = table, perm[b * slots:].contiguous()
        st["k"], st["v"] = normal(pool, page, hkv, d), normal(pool, page, hkv, d)
        st["pk"], st["pv"] = st["k"], st["v"]  # one pool holds the prefix and the sequences' own pages
        st["prefix_used"] = _int32([case["prefix"]])
    else:
        st["table"] = st["common"] = st["prefix_used"] = None
        st["k"], st["v"] = normal(b, case["max_len"], hkv, d), normal(b, case["max_len"], hkv, d)
        st["pk"], st["pv"] = normal(case["prefix"], hkv, d), normal(case["prefix"], hkv, d)
    return st


# ----------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "rotary":
        return _own_rotary(state) if own else _plain_rotary(state)
    if op == "append":
        return _own_append(state) if own else _plain_append(state)
    return _own_prefix(state) if own else _plain_prefix(state)


def _own_rotary(st):
    fsa, _ = _framework()
    case = st["case"]
    q, k = fsa.apply_rotary_func(st["q"], st["k"], st["cos"], st["sin"], cu_seqlens=st.get("cu"),
                                 interleaved=case["interleaved"])
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
    return q.detach(), k.detach(), dq, dk


def _own_append(st):
    _, kvcache = _framework()
    case, sc = st["case"], st["scales"] or (None, None, None)
    # a call that takes pages changes the table and the stack: each pass has its own
    used, table, count = st["used"], st["table"], st["count"]
    if case["alloc"]:
        used, table, count = used.clone(), table.clone(), count.clone()
    q = kvcache.append_kv_rotary(st["q"], st["k"], st["v"], st["kc"], st["vc"], used, st["cos"], st["sin"],
                                 page_table=table, free_pages=st["free"], free_count=count, cu_seqlens_new=st["cu"],
                                 seqlen_offsets=st["offset"], interleaved=case["interleaved"], query_scale=sc[0],
                                 key_scale=sc[1], value_scale=sc[2], advance=case["alloc"])
    return _append_outputs(st, q, used, table, count)


def _append_outputs(st, q, used, table, count):
    case, kc, vc = st["case"], st["kc"], st["vc"]
    if st["scales"]:
        # scales are powers of two: the products are exact
        q, kc, vc = (t.to(torch.bfloat16) * s.to(torch.bfloat16) for t, s in zip((q, kc, vc), st["scales"]))
    return (q, kc, vc, used, table, count) if case["alloc"] else (q, kc, vc)


def _own_prefix(st):
    fsa, _ = _framework()
    return fsa.flash_dense_attn_with_shared_prefix_func(
        st["q"], st["k"], st["v"], st["pk"], st["pv"], page_table=st["table"], seqused_k=st["used"],
        prefix_page_table=st["common"], prefix_seqused=st["prefix_used"], return_lse=True)


def _rotate(x, cos, sin, interleaved):
    """x [.., H, D] in fp32 and the rows of the tables that belong to its tokens [.., R / 2]."""
    half = cos.shape[-1]
    c, s = cos[..., None, :], sin[..., None, :]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * c - b * s
        y[..., 1:2 * half:2] = b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * c - b * s
        y[..., half:2 * half] = b * c + a * s
    return y


def _token_places(cu, total):
    """Packed tokens: the sequence of each and its place in it."""
    t = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    return b, t - cu.long()[b]


def _plain_rotary(st):
    case = st["case"]
    if case["packed"]:
        _, pos = _token_places(st["cu"], st["q"].shape[0])
    else:
        pos = torch.arange(case["seq"], device="cuda")
    cos, sin = st["cos"][pos], st["sin"][pos]
    dt = st["q"].dtype
    with torch.no_grad():
        return tuple(_rotate(x.float(), cos, s, case["interleaved"]).to(dt)
                     for x, s in ((st["q"], sin), (st["k"], sin), (st["gq"], -sin), (st["gk"], -sin)))


def _append_places(st, lengths):
    """The sequence, slot and rotary position of every new token, in the order of the rows."""
    case = st["case"]
    if case["packed"]:
        b, t = _token_places(st["cu"], st["q"].shape[0])
    else:
        t = torch.arange(case["new"], device="cuda").repeat(case["batch"])
        b = torch.arange(case["batch"], device="cuda").repeat_interleave(case["new"])
    slot = lengths.long()[b] + t
    return b, slot, slot + st["offset"]


def _take_pages(st, used, table, count, new):
    """Missing pages of the slots that receive rows, from the top of the stack, in the order of sequences and slots."""
    page = st["case"]["page"]
    first, last = used.long() // page, (used.long() + new - 1) // page
    i = torch.arange(table.shape[1], device="cuda")[None, :]
    missing = (table < 0) & (i >= first[:, None]) & (i <= last[:, None]) & (new[:, None] > 0)
    rank = missing.flatten().long().cumsum(0).view(table.shape)
    pages = st["free"][(count.long() - rank).clamp(min=0)]
    return torch.where(missing, pages, table), count - missing.sum().to(torch.int32)


def _plain_append(st):
    case = st["case"]
    used, table, count = st["used"], st["table"], st["count"]
    b, slot, pos = _append_places(st, used)
    if case["alloc"]:
        new = (st["cu"][1:] - st["cu"][:-1]).long() if case["packed"] else torch.full_like(used, case["new"]).long()
        table, count = _take_pages(st, used, table, count, new)
        used = used + new.to(torch.int32)
    cos, sin = st["cos"][pos], st["sin"][pos]
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    q = _rotate(st["q"].reshape(-1, hq, d).float(), cos, sin, case["interleaved"])
    k = _rotate(st["k"].reshape(-1, hkv, d).float(), cos, sin, case["interleaved"])
    v = st["v"].reshape(-1, hkv, d).float()
    q_dtype = st["q"].dtype
    if st["scales"]:
        top, q_dtype = _FP8_MAX[case["cache"]], st["kc"].dtype
        q, k, v = ((x / s).clamp(-top, top) for x, s in zip((q, k, v), st["scales"]))
    if case["page"]:
        where = (table[b, slot // case["page"]].long(), slot % case["page"])
    else:
        where = (b, slot)
    if st["scales"]:  # indexed stores of bytes
        st["kc"].view(torch.uint8)[where] = k.to(st["kc"].dtype).view(torch.uint8)
        st["vc"].view(torch.uint8)[where] = v.to(st["vc"].dtype).view(torch.uint8)
    else:
        st["kc"][where] = k.to(st["kc"].dtype)
        st["vc"][where] = v.to(st["vc"].dtype)
    return _append_outputs(st, q.to(q_dtype).view(st["q"].shape), used, table, count)


def _prefix_keys(st):
    """Prefix keys and values [P, Hkv, D] and the sequences' own [B, max_len, Hkv, D], as stored."""
    case = st["case"]
    if not case["page"]:
        return st["pk"], st["pv"], st["k"], st["v"]
    hkv, d = case["heads_kv"], case["head_dim"]
    common, table = st["common"].long(), st["table"].long()
    return (st["k"][common].reshape(-1, hkv, d)[:case["prefix"]], st["v"][common].reshape(-1, hkv, d)[:case["prefix"]],
            st["k"][table].reshape(case["batch"], -1, hkv, d), st["v"][table].reshape(case["batch"], -1, hkv, d))


def _plain_prefix(st):
    case = st["case"]
    hkv, d, b = case["heads_kv"], case["head_dim"], case["batch"]
    g = case["heads_q"] // hkv
    pk, pv, k, v = _prefix_keys(st)
    q = st["q"].float().view(b, hkv, g, d).transpose(0, 1) * d**-0.5                        # [Hkv, B, G, D]
    first = torch.matmul(q.reshape(hkv, b * g, d), pk.float().permute(1, 2, 0)).view(hkv, b, g, -1)
    second = torch.matmul(q, k.float().permute(2, 0, 3, 1))                                 # [Hkv, B, G, max_len]
    outside = torch.arange(k.shape[1], device="cuda")[None, :] >= st["used"].long()[:, None]
    second = second.masked_fill(outside[None, :, None, :], -math.inf)
    m = torch.maximum(first.amax(-1), second.amax(-1))
    first, second = (first - m[..., None]).exp(), (second - m[..., None]).exp()
    total = first.sum(-1) + second.sum(-1)
    out = torch.matmul(first.view(hkv, b * g, -1), pv.float().transpose(0, 1)).view(hkv, b, g, d)
    out = out + torch.matmul(second, v.float().permute(2, 0, 1, 3))
    out = (out / total[..., None]).transpose(0, 1).reshape(b, -1, d)
    lse = (m + total.log()).transpose(0, 1).reshape(b, -1)
    return out.to(st["q"].dtype), lse


# ----------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, interleaved, backwards=False):
    """Pairs as complex numbers, times cos + i sin (its conjugate for the gradient)."""
    r = 2 * cos.shape[-1]
    head = x[..., :r].double()
    pair = head.unflatten(-1, (r // 2, 2)) if interleaved else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pair.contiguous())
    w = torch.complex(cos.double(), -sin.double() if backwards else sin.double()).unsqueeze(-2)
    y = torch.view_as_real(z * w)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat([y, x[..., r:].double()], dim=-1)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "append": _exact_append, "prefix": _exact_prefix}[case["op"]](st)


def _exact_rotary(st):
    case = st["case"]
    if case["packed"]:
        pos = torch.cat([torch.arange(n) for n in _lengths(case, case["batch"], 1, case["seq"])]).cuda()
    else:
        pos = torch.arange(case["seq"], device="cuda").expand(case["batch"], -1)
    cos, sin, il = st["cos"][pos], st["sin"][pos], case["interleaved"]
    return (_turn(st["q"], cos, sin, il), _turn(st["k"], cos, sin, il), _turn(st["gq"], cos, sin, il, True),
            _turn(st["gk"], cos, sin, il, True))


def _nearest_fp8(x, name):
    """The nearest value of the format, halves to the even one; beyond the largest value that one."""
    bits, lowest = (3, -6) if name == "e4m3" else (2, -14)  # bits behind the point, exponent of the smallest normal value
    exponent = torch.frexp(x)[1].double().sub(1).clamp(min=lowest)
    step = torch.exp2(exponent - bits)
    return (torch.round(x / step) * step).clamp(-_FP8_MAX[name], _FP8_MAX[name])


def _exact_append(st):
    case = st["case"]
    new, used = _new_lengths(case), st["used"].tolist()
    table = st["table"].tolist() if case["page"] else None
    free = st["free"].tolist() if case["alloc"] else None
    count = int(st["count"]) if case["alloc"] else 0
    kc, vc = st["kc"].double(), st["vc"].double()
    if st["scales"]:
        kc, vc = kc * st["scales"][1].double(), vc * st["scales"][2].double()
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    q, k, v = st["q"].reshape(-1, hq, d), st["k"].reshape(-1, hkv, d), st["v"].reshape(-1, hkv, d).double()
    turned, row = [], 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        slots = list(range(used[b], used[b] + n))
        at = torch.tensor(slots, device="cuda") + st["offset"]
        rows = slice(row, row + n)
        row += n
        qb = _turn(q[rows], st["cos"][at], st["sin"][at], case["interleaved"])
        kb, vb = _turn(k[rows], st["cos"][at], st["sin"][at], case["interleaved"]), v[rows]
        if st["scales"]:
            qb, kb, vb = (_nearest_fp8(x / s.double(), case["cache"]) * s.double() for x, s in zip((qb, kb, vb), st["scales"]))
        turned.append(qb)
        if case["page"]:
            for i in range(slots[0] // case["page"], slots[-1] // case["page"] + 1):
                if table[b][i] < 0:
                    count -= 1
                    table[b][i] = free[count]
            line = torch.tensor([table[b][s // case["page"]] * case["page"] + s % case["page"] for s in slots], device="cuda")
            kc.view(-1, hkv, d)[line], vc.view(-1, hkv, d)[line] = kb, vb
        else:
            kc[b, slots[0]:slots[-1] + 1], vc[b, slots[0]:slots[-1] + 1] = kb, vb
    q = torch.cat(turned).view(st["q"].shape)
    if not case["alloc"]:
        return q, kc, vc
    return q, kc, vc, _int32([u + n for u, n in zip(used, new)]), _int32(table), _int32([count])


def _exact_prefix(st):
    case = st["case"]
    hkv, d, b = case["heads_kv"], case["head_dim"], case["batch"]
    g = case["heads_q"] // hkv
    pk, pv, k, v = _prefix_keys(st)
    lens = st["used"].tolist()
    out = torch.empty(b, case["heads_q"], d, dtype=torch.float64, device="cuda")
    lse = torch.empty(b, case["heads_q"], dtype=torch.float64, device="cuda")
    for h in range(hkv):
        keys, values = pk[:, h].double(), pv[:, h].double()
        for b0 in range(0, b, 64):  # scores of 64 sequences at a time
            q = st["q"][b0:b0 + 64, h * g:(h + 1) * g].double()
            n = q.shape[0]
            common = (q.reshape(n * g, d) @ keys.T / math.sqrt(d)).view(n, g, -1)
            alone = torch.einsum("bgd,bsd->bgs", q, k[b0:b0 + n, :, h].double()) / math.sqrt(d)
            seen = torch.arange(k.shape[1], device="cuda")[None, :] < _int32(lens[b0:b0 + n])[:, None]
            scores = torch.cat([common, alone.masked_fill(~seen[:, None, :], -math.inf)], dim=-1)
            z = torch.logsumexp(scores, dim=-1)
            p = torch.exp(scores - z[..., None])
            o = (p[..., :keys.shape[0]].reshape(n * g, -1) @ values).view(n, g, d)
            o = o + torch.einsum("bgs,bsd->bgd", p[..., keys.shape[0]:], v[b0:b0 + n, :, h].double())
            out[b0:b0 + n, h * g:(h + 1) * g], lse[b0:b0 + n, h * g:(h + 1) * g] = o, z
    return out, lse
