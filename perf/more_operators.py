"""Operators measured against their plain forms: rotary positions with several axes and their gradient, a key-value cache
whose rows are quantised as they are written and read back, and decode attention that reads such a cache.

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
_CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "int4": torch.uint8}


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
        # a training step of a layer over text and video: time, height and width share the pairs in three runs
        dict(name="axes-train", op="axes", packed=False, batch=4, seq=4096, heads_q=32, heads_kv=8, head_dim=128,
             rotary_dim=128, sections="16,24,24", dealt=False, interleaved=False, dtype="bf16"),
        # patches of images of many sizes in one packed row, two axes dealt out pair by pair
        dict(name="axes-patches", op="axes", packed=True, batch=1, seq=20011, heads_q=16, heads_kv=16, head_dim=80,
             rotary_dim=80, sections="20,20", dealt=True, interleaved=True, dtype="fp16"),
        # one short prompt with an odd length, where the launch is what counts
        dict(name="axes-short", op="axes", packed=False, batch=1, seq=77, heads_q=8, heads_kv=2, head_dim=64,
             rotary_dim=64, sections="12,10,10", dealt=True, interleaved=False, dtype="bf16"),
        # a decode step of a batch of young conversations, 8-bit rows, pages assigned by the scheduler
        dict(name="append-step", op="append", packed=False, batch=64, new=1, lens=3, max_len=31, page=32, alloc=False,
             heads_q=64, heads_kv=8, head_dim=128, rotary_dim=128, axes=False, interleaved=False, dtype="bf16",
             codes="int8", group=0, by_head=True),
        # prompt chunks with images in them, 4-bit rows, pages taken from the stack of free ones, read back for the prompt's attention
        dict(name="append-chunks", op="append", packed=True, batch=16, new=4000, lens=5, max_len=1500, page=64, alloc=True,
             heads_q=32, heads_kv=8, head_dim=128, rotary_dim=128, axes=True, interleaved=False, dtype="bf16",
             codes="int4", group=64, by_head=True),
        # a long conversation, 8-bit pages: its keys and values in 16 bits in front of the next prompt
        dict(name="read-prompt", op="read", packed=True, batch=8, lens=7, max_len=16000, page=64, heads_kv=8, head_dim=128,
             dtype="bf16", codes="int8", group=0, by_head=True),
        # a few short rows, 4 bits in groups of 32, contiguous
        dict(name="read-few", op="read", packed=False, batch=5, lens=9, max_len=333, page=0, heads_kv=4, head_dim=96,
             dtype="fp16", codes="int4", group=32, by_head=False),
        # one user, one token, a short contiguous cache: latency
        dict(name="decode-one", op="decode", batch=1, lens=2, max_len=2001, page=0, topk=0, heads_q=16, heads_kv=4,
             head_dim=64, dtype="fp16", codes="int8", group=0, by_head=True),
        # a chat service: 64 conversations of unequal length, 8-bit pages of 64
        dict(name="decode-chat", op="decode", batch=64, lens=4, max_len=8192, page=64, topk=0, heads_q=32, heads_kv=8,
             head_dim=128, dtype="bf16", codes="int8", group=0, by_head=True),
        # long documents in 4 bits, groups of 64 columns
        dict(name="decode-long", op="decode", batch=8, lens=6, max_len=100000, page=128, topk=0, heads_q=64, heads_kv=8,
             head_dim=128, dtype="bf16", codes="int4", group=64, by_head=True),
        # sparse decode: 2048 chosen positions of each sequence, FP8 rows with their own scales
        dict(name="decode-topk", op="decode", batch=32, lens=8, max_len=32768, page=256, topk=2048, heads_q=32, heads_kv=4,
             head_dim=128, dtype="bf16", codes="e4m3", group=0, by_head=True),
        # odd everything: five query heads per KV head, head size 96, 4 bits in groups of 32, heads side by side in a page
        dict(name="decode-odd", op="decode", batch=37, lens=9, max_len=3333, page=32, topk=0, heads_q=20, heads_kv=4,
             head_dim=96, dtype="fp16", codes="int4", group=32, by_head=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_sections(rng, pairs):
    """A division of the pairs among two to four axes, and whether they are dealt out one by one."""
    axes = rng.choice([2, 3, 3, 4])
    if rng.random() < 0.4 and pairs >= 2 * axes:
        share = [rng.randint(1, pairs // axes) for _ in range(axes - 1)]
        return [pairs - sum(share)] + share, True
    unit = 8 if pairs % 8 == 0 and pairs >= 8 * axes and rng.random() < 0.6 else 1
    cuts = sorted(rng.sample(range(1, pairs // unit), axes - 1))
    return [unit * (b - a) for a, b in zip([0] + cuts, cuts + [pairs // unit])], False


def draw(rng):
    op = rng.choice(["axes", "append", "read", "decode", "decode"])
    dtype = rng.choice(["bf16", "fp16"])
    heads_kv = rng.choice([1, 2, 3, 4, 8])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
    lens = rng.randrange(1, 1 << 30)
    if op == "axes":
        head_dim = rng.choice([32, 48, 64, 80, 96, 112, 128])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
        packed = rng.random() < 0.5
        batch = 1 if packed else _log_int(rng, 1, 32)
        seq = max(1, min(_log_int(rng, 1, 20000), 80_000_000 // (batch * (heads_q + heads_kv) * head_dim)))
        sections, dealt = _draw_sections(rng, rotary_dim // 2)
        return dict(op=op, packed=packed, batch=batch, seq=seq, heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim,
                    rotary_dim=rotary_dim, sections=",".join(map(str, sections)), dealt=dealt,
                    interleaved=rng.random() < 0.4, dtype=dtype)
    codes = rng.choice(["int8", "int8", "e4m3", "int4", "int4"])
    if codes == "int4":
        head_dim = rng.choice([32, 64, 96, 128, 128])
        group = 64 if head_dim % 64 == 0 and rng.random() < 0.6 else 32
    else:
        head_dim, group = rng.choice([32, 48, 64, 80, 96, 112, 128, 128]), 0
    page = rng.choice([0, 32, 64, 128, 256])
    by_head = rng.random() < 0.7
    if op == "append":
        packed = rng.random() < 0.5
        batch = _log_int(rng, 1, 128)
        new = rng.choice([1, 1, rng.randint(2, 8), max(1, min(_log_int(rng, 9, 4000), 32000 // batch))])
        rotary_dim = rng.choice([head_dim, head_dim, 32, 0])
        return dict(op=op, packed=packed, batch=batch, new=new, lens=lens, max_len=_log_int(rng, 1, 60 if new < 9 else 1500),
                    page=page, alloc=page > 0 and rng.random() < 0.5, heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim,
                    rotary_dim=rotary_dim, axes=rotary_dim > 0 and rng.random() < 0.5, interleaved=rng.random() < 0.4,
                    dtype=dtype, codes=codes, group=group, by_head=by_head)
    if op == "read":
        batch = _log_int(rng, 1, 64)
        max_len = max(1, min(_log_int(rng, 1, 100000), 130_000_000 // (batch * heads_kv * head_dim)))
        return dict(op=op, packed=rng.random() < 0.5, batch=batch, lens=lens, max_len=max_len, page=page, heads_kv=heads_kv,
                    head_dim=head_dim, dtype=dtype, codes=codes, group=group, by_head=by_head)
    batch = _log_int(rng, 1, 256)
    max_len = max(1, min(_log_int(rng, 1, 131072), 400_000_000 // (batch * heads_kv * head_dim), 80_000_000 // (batch * heads_q)))
    topk = min(max_len, _log_int(rng, 1, 4096)) if rng.random() < 0.3 else 0
    return dict(op=op, batch=batch, lens=lens, max_len=max_len, page=page, topk=topk, heads_q=heads_q, heads_kv=heads_kv,
                head_dim=head_dim, dtype=dtype, codes=codes, group=group, by_head=by_head)


def _lengths(case, count, low, high, salt=0):
    """Unequal lengths that belong to the case (not to the seed): the first is the largest, one is the smallest."""
    rng = random.Random(case["lens"] * 7919 + salt)
    out = [high] + [rng.randint(low, high) for _ in range(count - 1)]
    if count > 2:
        out[rng.randrange(1, count)] = low
    return out


def _new_lengths(case):
    return _lengths(case, case["batch"], min(1, case["new"]), case["new"], 1) if case["packed"] else [case["new"]] * case["batch"]


def _row_bytes(case):
    """Codes and scales of one (token, head) row."""
    d = case["head_dim"]
    return d // 2 + 4 * (d // case["group"]) if case["codes"] == "int4" else d + 4


def work(case):
    d, hkv = case["head_dim"], case["heads_kv"]
    if case["op"] == "axes":
        elems = case["batch"] * case["seq"] * (case["heads_q"] + hkv) * d
        axes = len(case["sections"].split(","))
        tokens = case["batch"] * case["seq"]
        # forward and gradient: each reads and writes every element once
        return {"bytes": 4 * elems * 2 + 2 * tokens * axes * 4, "flops": 2 * 3 * elems * case["rotary_dim"] // d}
    if case["op"] == "append":
        new, used = sum(_new_lengths(case)), sum(_lengths(case, case["batch"], 0, case["max_len"], 2))
        q, kv, row = new * case["heads_q"] * d, new * hkv * d, _row_bytes(case)
        # the new rows turned and quantised, then everything that the cache holds read back
        turned = 2 * q * 2 if case["rotary_dim"] else 0
        return {"bytes": turned + 2 * kv * 2 + 2 * new * hkv * row + 2 * (new + used) * hkv * (row + 2 * d),
                "flops": 3 * (q + kv) * case["rotary_dim"] // d + 6 * kv + 4 * (new + used) * hkv * d}
    if case["op"] == "read":
        tokens = sum(_lengths(case, case["batch"], 0, case["max_len"]))
        return {"bytes": 2 * tokens * hkv * (_row_bytes(case) + 2 * d), "flops": 4 * tokens * hkv * d}
    keys = _keys(case)
    rows = case["batch"] * case["heads_q"]
    return {"bytes": 2 * keys * hkv * _row_bytes(case) + 2 * rows * d * 2 + 4 * rows + (4 * case["batch"] * case["topk"]),
            "flops": 4 * d * case["heads_q"] * keys}


def _keys(case):
    """Keys that a decode reads: all that are there, or the chosen ones."""
    lens = _lengths(case, case["batch"], 0, case["max_len"])
    return sum(min(n, case["topk"]) for n in lens) if case["topk"] else sum(lens)


# ----------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------
def _tables(positions, rotary_dim):
    """cos and sin of position * 10000^(-2i / R): angles in 64 bits, kept in 32."""
    freq = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cuda") / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _int32(out)


def _grid_positions(place, axes):
    """Positions of tokens at `place` on every axis: text counts on all alike; every other run of 256 tokens is an image of
    16 x 16, one moment in time."""
    image = (place // 256) % 2 == 1
    start, inside = place // 256 * 256, place % 256
    rows = [place, start + inside // 16, start + inside % 16, place % 97]
    rows[0] = torch.where(image, start, place)
    return torch.stack([torch.where(image, r, place) if i else r for i, r in enumerate(rows[:axes])]).to(torch.int32)


def _sections(case):
    if case["op"] == "axes":
        return [int(n) for n in case["sections"].split(",")]
    pairs = case["rotary_dim"] // 2
    return [pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8]  # time, height, width


def _storage(case, blocks, size, gen):
    """A cache [blocks, size, heads, ..] with rows in it: codes of normal values, and their scales."""
    d, hkv, codes = case["head_dim"], case["heads_kv"], case["codes"]

    def make(width, *more, fill):
        if case["by_head"]:  # each head's rows of a block side by side in memory
            return fill((blocks, hkv, size, width) + more).transpose(1, 2)
        return fill((blocks, size, hkv, width) + more)

    def normal(shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if codes == "int4":
        def code(shape):
            out = torch.empty(shape, dtype=torch.uint8, device="cuda")
            for i in range(0, shape[0], 1 << 12):  # bounds what the random numbers take
                part = out[i:i + (1 << 12)]
                lo, hi = (normal(part.shape).mul_(3.2).add_(8).round_().clamp_(0, 15).to(torch.uint8) for _ in range(2))
                part.copy_(lo + 16 * hi)
            return out

        def scale(shape):
            s = torch.rand(shape[:-1], generator=gen, device="cuda") * 0.2 + 0.2
            z = normal(shape[:-1]) * 0.1
            return torch.stack([s, z], dim=-1).to(torch.bfloat16)

        return make(d // 2, fill=code), make(d // case["group"], 2, fill=scale)

    def code(shape):
        out = torch.empty(shape, dtype=_CODES[codes], device="cuda")
        for i in range(0, shape[0], 1 << 12):
            x = normal(out[i:i + (1 << 12)].shape)
            x = x.mul_(46.0).round_().clamp_(-127, 127) if codes == "int8" else x.mul_(160.0).clamp_(-448, 448)
            out.view(torch.uint8)[i:i + (1 << 12)] = x.to(out.dtype).view(torch.uint8)
        return out

    top = 127.0 if codes == "int8" else 448.0
    return make(d, fill=code), make(1, fill=lambda s: (torch.rand(s, generator=gen, device="cuda") + 2.2) / top)


def _cache(st, case, capacity, gen):
    """Codes and scales of keys and values, contiguous or in scattered pages."""
    b = case["batch"]
    if case["page"]:
        slots = -(-capacity // case["page"])
        blocks, size = b * slots + 3, case["page"]
        perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        st["table"], st["perm"] = perm[: b * slots].view(b, slots).contiguous(), perm
    else:
        blocks, size, st["table"] = b, capacity, None
    st["k"], st["ks"] = _storage(case, blocks, size, gen)
    st["v"], st["vs"] = _storage(case, blocks, size, gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    hkv, d, b = case["heads_kv"], case["head_dim"], case["batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    st = {"case": case}
    if case["op"] == "axes":
        lead = (case["seq"],) if case["packed"] else (b, case["seq"])
        place = torch.arange(case["seq"], device="cuda").expand(lead)
        shift = 0 if case["packed"] else torch.arange(b, device="cuda")[:, None] * 5
        st["ids"] = _grid_positions(place + shift, len(_sections(case)))
        st["cos"], st["sin"] = _tables(case["seq"] + 5 * b + 256, case["rotary_dim"])
        hq = case["heads_q"]
        st["q"], st["k"] = normal(*lead, hq, d).requires_grad_(), normal(*lead, hkv, d).requires_grad_()
        st["gq"], st["gk"] = normal(*lead, hq, d), normal(*lead, hkv, d)
        return st
    if case["op"] == "append":
        new, used = _new_lengths(case), _lengths(case, b, 0, case["max_len"], 2)
        after = [n + u for n, u in zip(new, used)]
        lead = (sum(new),) if case["packed"] else (b, case["new"])
        st["cu"] = _cumulative(new) if case["packed"] else None
        st["q"] = normal(*lead, case["heads_q"], d) if case["rotary_dim"] else None
        st["kn"], st["vn"] = normal(*lead, hkv, d), normal(*lead, hkv, d)
        capacity = case["max_len"] + case["new"]
        st["capacity"] = capacity
        st["used"], st["after"], st["cu_after"] = _int32(used), _int32(after), _cumulative(after)
        st["total"] = sum(after)
        st["cos"] = st["sin"] = st["ids"] = None
        if case["rotary_dim"]:
            st["cos"], st["sin"] = _tables(capacity + 256, case["rotary_dim"])
        if case["axes"]:
            place = torch.cat([torch.arange(u, u + n) for u, n in zip(used, new)]).cuda().view(lead)
            st["ids"] = _grid_positions(place, 3)
        _cache(st, case, capacity, gen)
        st["free"] = st["count"] = None
        if case["alloc"]:
            # only the pages that hold something are assigned; the rest is on the stack
            perm, slots = st["perm"], st["table"].shape[1]
            held = (st["used"].long() + case["page"] - 1) // case["page"]
            st["table"] = torch.where(torch.arange(slots, device="cuda")[None, :] < held[:, None], st["table"], -1).to(torch.int32)
            flags = torch.zeros(perm.numel(), dtype=torch.bool, device="cuda")
            flags[st["table"][st["table"] >= 0].long()] = True
            free = perm.flip(0)
            order = torch.argsort(flags[free.long()].int(), stable=True)
            st["free"] = free[order].contiguous()
            st["count"] = (perm.numel() - flags.sum()).to(torch.int32).reshape(1)
        return st
    lens = _lengths(case, b, 0, case["max_len"])
    st["used"] = _int32(lens)
    _cache(st, case, case["max_len"], gen)
    if case["op"] == "read":
        st["cu"], st["total"] = _cumulative(lens), sum(lens)
        return st
    st["q"] = normal(b, case["heads_q"], d)
    st["at"] = None
    if case["topk"]:
        # chosen positions in ascending order; what a short sequence does not have is -1
        scores = torch.rand(b, case["max_len"], generator=gen, device="cuda")
        scores.masked_fill_(torch.arange(case["max_len"], device="cuda")[None, :] >= st["used"][:, None], -1.0)
        at = scores.topk(case["topk"], dim=1).indices.sort(dim=1).values
        st["at"] = torch.where(at < st["used"][:, None], at, -1).to(torch.int32)
    return st


# ----------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "axes":
        return _own_axes(state) if own else _plain_axes(state)
    if op == "append":
        return _own_append(state) if own else _plain_append(state)
    if op == "read":
        return _own_read(state) if own else _plain_read(state)
    return _own_decode(state) if own else _plain_decode(state)


def _own_axes(st):
    fsa, _ = _framework()
    case = st["case"]
    q, k = fsa.apply_rotary_axes_func(st["q"], st["k"], st["cos"], st["sin"], st["ids"], _sections(case),
                                      axes_dealt=case["dealt"], interleaved=case["interleaved"])
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
    return q.detach(), k.detach(), dq, dk


def _own_append(st):
    _, kvcache = _framework()
    case = st["case"]
    # a call that takes pages changes the table and the stack: each pass has its own
    used, table, count = st["used"], st["table"], st["count"]
    if case["alloc"]:
        used, table, count = used.clone(), table.clone(), count.clone()
    q = kvcache.append_kv_quantized(st["q"], st["kn"], st["vn"], st["k"], st["v"], st["ks"], st["vs"], used, st["cos"], st["sin"],
                                    page_table=table, free_pages=st["free"], free_count=count, cu_seqlens_new=st["cu"],
                                    position_ids=st["ids"], sections=_sections(case) if case["axes"] else None,
                                    interleaved=case["interleaved"], advance=case["alloc"])
    if case["packed"]:
        k, v = kvcache.read_kv_quantized(st["k"], st["v"], st["ks"], st["vs"], st["after"], page_table=table,
                                         cu_seqlens=st["cu_after"], total=st["total"], dtype=st["kn"].dtype)
    else:
        k, v = kvcache.read_kv_quantized(st["k"], st["v"], st["ks"], st["vs"], st["after"], page_table=table,
                                         max_seqlen=st["capacity"], dtype=st["kn"].dtype)
    out = [k, v] if q is None else [q, k, v]
    return out + [used, table, count] if case["alloc"] else out


def _own_read(st):
    _, kvcache = _framework()
    case = st["case"]
    rows = dict(cu_seqlens=st["cu"], total=st["total"]) if case["packed"] else dict(max_seqlen=case["max_len"])
    return kvcache.read_kv_quantized(st["k"], st["v"], st["ks"], st["vs"], st["used"], page_table=st["table"],
                                     dtype=_DTYPES[case["dtype"]], **rows)


def _own_decode(st):
    fsa, _ = _framework()
    return fsa.flash_dense_attn_with_quantized_kvcache_func(
        st["q"], st["k"], st["v"], st["ks"], st["vs"], page_table=st["table"], gather_kv_indices=st["at"],
        seqused_k=st["used"], return_lse=True)


# ----------------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------------
def _axis_of_pairs(sections, dealt):
    """The axis of every pair: run after run, or dealt out in turn while an axis has pairs left, the rest to the first."""
    pairs, axes = sum(sections), len(sections)
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % axes if i // axes < sections[i % axes] else 0 for i in range(pairs)]


def _angles(st, ids, sections, dealt):
    """Rows of the tables [.., R / 2] whose columns come from the positions of their axes."""
    axis = torch.tensor(_axis_of_pairs(sections, dealt), device="cuda")
    c, s = st["cos"][ids[0].long()], st["sin"][ids[0].long()]
    for a in range(1, len(sections)):
        c = torch.where(axis == a, st["cos"][ids[a].long()], c)
        s = torch.where(axis == a, st["sin"][ids[a].long()], s)
    return c, s


def _rotate(x, cos, sin, interleaved):
    """x [.., H, D] in fp32 and the angles of its tokens [.., R / 2]."""
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


def _plain_axes(st):
    case = st["case"]
    cos, sin = _angles(st, st["ids"], _sections(case), case["dealt"])
    dt = st["q"].dtype
    with torch.no_grad():
        return tuple(_rotate(x.float(), cos, s, case["interleaved"]).to(dt)
                     for x, s in ((st["q"], sin), (st["k"], sin), (st["gq"], -sin), (st["gk"], -sin)))


def _quantise(x, case):
    """Rows [.., D] in fp32 -> codes and scales as they are kept."""
    if case["codes"] == "int4":
        g = x.unflatten(-1, (-1, case["group"]))
        low, high = g.amin(-1), g.amax(-1)
        s = ((high - low) / 15).to(torch.bfloat16)
        z = (low + 8 * s.float()).to(torch.bfloat16)
        inverse = torch.where(s > 0, 1 / s.float(), 0)
        n = (((g - z.float()[..., None]) * inverse[..., None]).round() + 8).clamp(0, 15).to(torch.uint8).flatten(-2)
        return n[..., 0::2] + 16 * n[..., 1::2], torch.stack([s, z], dim=-1)
    top = 127.0 if case["codes"] == "int8" else 448.0
    s = x.abs().amax(-1, keepdim=True) / top
    n = (x * torch.where(s > 0, 1 / s, 0)).clamp(-top, top)
    return (n.round() if case["codes"] == "int8" else n).to(_CODES[case["codes"]]), s


def _values(codes, scales):
    """What codes and scales stand for, in fp32."""
    if codes.dtype != torch.uint8:
        return codes.float() * scales
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float() - 8
    n = n.unflatten(-1, (scales.shape[-2], -1))
    return (n * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2)


def _token_places(cu, total):
    """Packed tokens: the sequence of each and its place in it."""
    t = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    return b, t - cu.long()[b]


def _where(case, table, b, slot):
    """Indices of a cache's rows."""
    return (table[b, slot // case["page"]].long(), slot % case["page"]) if case["page"] else (b, slot)


def _take_pages(st, used, table, count, new):
    """Missing pages of the slots that receive rows, from the top of the stack, in the order of sequences and slots."""
    page = st["case"]["page"]
    first, last = used.long() // page, (used.long() + new - 1) // page
    i = torch.arange(table.shape[1], device="cuda")[None, :]
    missing = (table < 0) & (i >= first[:, None]) & (i <= last[:, None]) & (new[:, None] > 0)
    rank = missing.flatten().long().cumsum(0).view(table.shape)
    pages = st["free"][(count.long() - rank).clamp(min=0)]
    return torch.where(missing, pages, table), count - missing.sum().to(torch.int32)


def _put(cache, where, rows):
    if cache.dtype == torch.float8_e4m3fn:  # indexed stores of bytes
        cache, rows = cache.view(torch.uint8), rows.view(torch.uint8)
    cache[where] = rows


def _plain_append(st):
    case = st["case"]
    used, table, count = st["used"], st["table"], st["count"]
    hkv, d = case["heads_kv"], case["head_dim"]
    if case["packed"]:
        b, t = _token_places(st["cu"], st["kn"].shape[0])
    else:
        t = torch.arange(case["new"], device="cuda").repeat(case["batch"])
        b = torch.arange(case["batch"], device="cuda").repeat_interleave(case["new"])
    slot = used.long()[b] + t
    if case["alloc"]:
        new = (st["cu"][1:] - st["cu"][:-1]).long() if case["packed"] else torch.full_like(used, case["new"]).long()
        table, count = _take_pages(st, used, table, count, new)
        used = used + new.to(torch.int32)
    k, v = (x.reshape(-1, hkv, d).float() for x in (st["kn"], st["vn"]))
    q = st["q"]
    if case["rotary_dim"]:
        if case["axes"]:
            cos, sin = _angles(st, st["ids"].flatten(1), _sections(case), False)
        else:
            cos, sin = st["cos"][slot], st["sin"][slot]
        k = _rotate(k, cos, sin, case["interleaved"])
        q = _rotate(q.reshape(-1, case["heads_q"], d).float(), cos, sin, case["interleaved"]).to(q.dtype).view(q.shape)
    where = _where(case, table, b, slot)
    for x, codes, scales in ((k, st["k"], st["ks"]), (v, st["v"], st["vs"])):
        n, s = _quantise(x, case)
        _put(codes, where, n)
        scales[where] = s
    if case["packed"]:
        k, v = _plain_rows(st, table, st["cu_after"], st["total"], st["kn"].dtype)
    else:
        k, v = _plain_padded(st, table, st["after"], st["capacity"], st["kn"].dtype)
    out = [k, v] if q is None else [q, k, v]
    return out + [used, table, count] if case["alloc"] else out


def _plain_rows(st, table, cu, total, dtype):
    where = _where(st["case"], table, *_token_places(cu, total))
    return [_values(_take(c, where), s[where]).to(dtype) for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"]))]


def _take(cache, where):
    if cache.dtype == torch.float8_e4m3fn:
        return cache.view(torch.uint8)[where].view(cache.dtype)
    return cache[where]


def _plain_padded(st, table, used, length, dtype):
    case = st["case"]
    slot = torch.arange(length, device="cuda").repeat(case["batch"])
    b = torch.arange(case["batch"], device="cuda").repeat_interleave(length)
    inside = (slot < used.long()[b]).view(case["batch"], length, 1, 1)
    if case["page"]:
        table = table.clamp(min=0)  # slots without a page are outside
    where = _where(case, table, b, slot)
    out = []
    for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"])):
        x = _values(_take(c, where), s[where]).view(case["batch"], length, case["heads_kv"], case["head_dim"])
        out.append(torch.where(inside, x, 0).to(dtype))
    return out


def _plain_read(st):
    case = st["case"]
    dtype = _DTYPES[case["dtype"]]
    if case["packed"]:
        return _plain_rows(st, st["table"], st["cu"], st["total"], dtype)
    return _plain_padded(st, st["table"], st["used"], case["max_len"], dtype)


def _decode_places(st):
    """Sequence and slot of every key that may be attended to [B, n], and whether it is."""
    case = st["case"]
    if case["topk"]:
        slot = st["at"].long()
    else:
        slot = torch.arange(case["max_len"], device="cuda").expand(case["batch"], -1)
    inside = (slot >= 0) & (slot < st["used"].long()[:, None])
    b = torch.arange(case["batch"], device="cuda")[:, None].expand_as(slot)
    return b, slot.clamp(min=0), inside


def _plain_decode(st):
    case = st["case"]
    hkv, d, b = case["heads_kv"], case["head_dim"], case["batch"]
    rows, slot, inside = _decode_places(st)
    where = _where(case, st["table"], rows, slot)
    k = _values(_take(st["k"], where), st["ks"][where]).permute(0, 2, 3, 1)  # [B, Hkv, D, n]
    q = st["q"].float().view(b, hkv, -1, d) * d**-0.5
    scores = torch.matmul(q, k).masked_fill(~inside[:, None, None, :], -math.inf)
    del k
    m = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(m == -math.inf, 0, m)).exp()
    total = p.sum(-1, keepdim=True)
    v = _values(_take(st["v"], where), st["vs"][where]).permute(0, 2, 1, 3)
    out = torch.matmul(p, v) / torch.where(total == 0, 1, total)
    lse = (m + total.log()).view(b, -1)
    return out.view(b, -1, d).to(st["q"].dtype), lse


# ----------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"axes": _exact_axes, "append": _exact_append, "read": _exact_read, "decode": _exact_decode}[case["op"]](st)


def _turn(x, angle, interleaved, backwards=False):
    """Pairs as complex numbers, times `angle` [.., R / 2] = cos + i sin (its conjugate for the gradient)."""
    r = 2 * angle.shape[-1]
    head = x[..., :r].double()
    pair = head.unflatten(-1, (r // 2, 2)) if interleaved else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_complex(pair.contiguous())
    y = torch.view_as_real(z * (angle.conj() if backwards else angle).unsqueeze(-2))
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat([y, x[..., r:].double()], dim=-1)


def _exact_angle(st, ids, sections, dealt):
    """One column at a time: the position of its axis."""
    columns, left, runs = [], list(sections), [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(sum(sections)):
        a = runs[i]
        if dealt:
            a = i % len(sections)
            if i // len(sections) >= sections[a]:
                a = 0
        left[a] -= 1
        at = ids[a].long()
        columns.append(torch.complex(st["cos"][at, i].double(), st["sin"][at, i].double()))
    assert left == [0] * len(sections)
    return torch.stack(columns, dim=-1)


def _exact_axes(st):
    case, il = st["case"], st["case"]["interleaved"]
    w = _exact_angle(st, st["ids"], _sections(case), case["dealt"])
    return _turn(st["q"], w, il), _turn(st["k"], w, il), _turn(st["gq"], w, il, True), _turn(st["gk"], w, il, True)


def _bf16(x):
    """The nearest value with eight significant bits, halves to the even one."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256), e - 8)


def _exact_values(x, case):
    """The values that stand for rows [.., D] after quantising."""
    if case["codes"] == "int4":
        g = x.reshape(*x.shape[:-1], -1, case["group"])
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        s = _bf16((high - low) / 15)
        z = _bf16(low + 8 * s)
        n = torch.round((g - z) / torch.where(s == 0, 1, s)).clamp(-8, 7)
        return (z + n * s).reshape(x.shape)
    top = 127.0 if case["codes"] == "int8" else 448.0
    s = x.abs().max(-1, keepdim=True).values / top
    y = x / torch.where(s == 0, 1, s)
    if case["codes"] == "int8":
        return torch.round(y) * s
    # three bits behind the point, smallest normal value 2^-6
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-top, top) * s


def _stored_values(codes, scales):
    """Values of kept rows, by columns."""
    if codes.dtype != torch.uint8:
        return codes.double() * scales.double()
    out = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    per = out.shape[-1] // scales.shape[-2]
    s = scales.double().repeat_interleave(per, dim=-2)
    return (out - 8) * s[..., 0] + s[..., 1]


def _sequence_values(st, table, codes, scales, b, n):
    """Values of the first n rows of sequence b [n, Hkv, D]."""
    page = st["case"]["page"]
    if not page:
        return _stored_values(codes[b, :n], scales[b, :n])
    pages = torch.tensor(table[b][:-(-n // page)], dtype=torch.long, device="cuda")
    kept = codes.view(torch.uint8)[pages].view(codes.dtype) if codes.dtype == torch.float8_e4m3fn else codes[pages]
    return _stored_values(kept.flatten(0, 1)[:n], scales[pages].flatten(0, 1)[:n])


def _laid_out(parts, lens, packed, length):
    if packed:
        return torch.cat(parts)
    out = torch.zeros((len(lens), length) + parts[0].shape[1:], dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        out[b, :n] = parts[b]
    return out


def _exact_read(st):
    case = st["case"]
    lens, table = st["used"].tolist(), st["table"].tolist() if case["page"] else None
    return [_laid_out([_sequence_values(st, table, c, s, b, n) for b, n in enumerate(lens)], lens, case["packed"], case["max_len"])
            for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"]))]


def _exact_append(st):
    case = st["case"]
    new, used = _new_lengths(case), st["used"].tolist()
    table = st["table"].tolist() if case["page"] else None
    free = st["free"].tolist() if case["alloc"] else None
    count = int(st["count"]) if case["alloc"] else 0
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["head_dim"]
    kn, vn = st["kn"].reshape(-1, hkv, d), st["vn"].reshape(-1, hkv, d)
    ids = st["ids"].flatten(1) if case["axes"] else None
    q, keys, values, row = [], [], [], 0
    for b, n in enumerate(new):
        old = [_sequence_values(st, table, c, s, b, used[b]) for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"]))]
        rows = slice(row, row + n)
        row += n
        k, v = kn[rows].double(), vn[rows].double()
        if case["rotary_dim"]:
            if case["axes"]:
                w = _exact_angle(st, ids[:, rows], _sections(case), False)
            else:
                at = torch.arange(used[b], used[b] + n, device="cuda")
                w = torch.complex(st["cos"][at].double(), st["sin"][at].double())
            k = _turn(kn[rows], w, case["interleaved"])
            q.append(_turn(st["q"].reshape(-1, hq, d)[rows], w, case["interleaved"]))
        if case["alloc"] and n:
            for i in range(used[b] // case["page"], (used[b] + n - 1) // case["page"] + 1):
                if table[b][i] < 0:
                    count -= 1
                    table[b][i] = free[count]
        keys.append(torch.cat([old[0], _exact_values(k, case)]))
        values.append(torch.cat([old[1], _exact_values(v, case)]))
    lens = [n + u for n, u in zip(new, used)]
    out = [_laid_out(x, lens, case["packed"], st["capacity"]) for x in (keys, values)]
    if case["rotary_dim"]:
        out = [torch.cat(q).view(st["q"].shape)] + out
    return out + [_int32(lens), _int32(table), _int32([count])] if case["alloc"] else out


def _exact_decode(st):
    case = st["case"]
    hkv, d, b = case["heads_kv"], case["head_dim"], case["batch"]
    lens, table = st["used"].tolist(), st["table"].tolist() if case["page"] else None
    out = torch.zeros(b, case["heads_q"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, case["heads_q"]), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k = _sequence_values(st, table, st["k"], st["ks"], i, n)
        v = _sequence_values(st, table, st["v"], st["vs"], i, n)
        if case["topk"]:
            at = st["at"][i][st["at"][i] >= 0].long()
            k, v = k[at], v[at]
        q = st["q"][i].double().view(hkv, -1, d)
        scores = torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(d)
        z = torch.logsumexp(scores, dim=-1)
        out[i] = torch.einsum("hgn,nhd->hgd", torch.exp(scores - z[..., None]), v).reshape(-1, d)
        lse[i] = z.reshape(-1)
    return out, lse
