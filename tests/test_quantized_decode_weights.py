"""Decode over a cache whose rows carry their own scales, where keys weigh very differently: what a key adds to the result is its
probability times its value, and neither of the two says by itself how finely it has to be held. Against 64 bits, relative to the
size of the result alone."""

import math

import pytest
import torch

from test_quantized_decode import FORMS, reference
from test_quantized_kvcache import KINDS, make_cache, quantised, values
from test_rotary import done, normal

DEV = "cuda"
FEW = [f for f in FORMS if f[1] in (64, 96, 128)]


def stored(x, kind, group):
    """Rows [B, H, n, D] -> codes and scales [B, n, H, ..] with a head's rows side by side, and their values in 64 bits [B, H, n, D]."""
    codes, scales = quantised(x, kind, group)
    if kind == "int4":
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double().unflatten(-1, (scales.shape[-2], -1)) - 8
        v = (n * scales[..., :1].double() + scales[..., 1:].double()).flatten(-2)
    else:
        v = codes.float().double() * scales.double()
    assert codes.dtype == KINDS[kind]
    return codes.transpose(1, 2), scales.transpose(1, 2), v


def attend(q, xk, xv, kind, group, scale):
    """The operator on the rows' quantised form, and in 64 bits: result, log-sum-exp, sum |p v|, sum |q k| of the largest score."""
    import flash_sparse_attn as fsa

    (ck, sk, k), (cv, sv, v) = stored(xk, kind, group), stored(xv, kind, group)
    out, lse = fsa.flash_dense_attn_with_quantized_kvcache_func(q, ck, cv, sk, sv, softmax_scale=scale, return_lse=True)
    done()
    b, h = k.shape[:2]
    qq = q.double().view(b, h, -1, q.shape[-1])
    s = qq @ k.transpose(-1, -2) * scale
    p = torch.softmax(s, -1)
    ref, size = ((p @ x).view(q.shape) for x in (v, v.abs()))
    reach = (qq.abs() @ k.abs().transpose(-1, -2)).amax() * scale
    return out.double(), lse.double(), ref, torch.logsumexp(s, -1).view(lse.shape), size, reach.item()


def score_error(d, reach):
    """How far a probability is off: scores are sums of D products in fp32 (4-bit rows: of codes and centres apart, at most three times as large), twice
    (numerator and sum), and 2^-19 for exponentials and the joining of parts."""
    return 2 * d * 2.0**-24 * 3 * reach + 2.0**-19


def rows_close(out, ref, dtype, extra, columns=slice(None)):
    """Rows as vectors. Their roundings are independent, and columns are sums of many keys: what rounding a probability times a scale to fp16 (2^-11,
    bf16 results alone) takes from each key adds up like the result itself does. The result is rounded once, below the normal numbers to their step."""
    info = torch.finfo(dtype)
    out, ref = out[..., columns], ref[..., columns]
    part = info.eps / 2 + (2.0**-11 if dtype == torch.bfloat16 else 0.0) + extra
    floor = info.smallest_normal * info.eps / 2 * math.sqrt(ref.shape[-1])
    off = (out - ref).norm(dim=-1) - floor
    assert (off <= part * ref.norm(dim=-1)).all(), f"{(off / ref.norm(dim=-1)).max().item():.3g} of the result, allowed {part:.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,d,group", FEW)
@pytest.mark.parametrize("per,n", [(2, 256), (12, 70), (3, 3000)])
def test_a_large_value_that_nobody_attends_to(kind, d, group, dtype, per, n):
    """One row 2^24 times the others' size, 2^-60 of their probability: first, in the middle and last. Relative to sum |p v| in every column: a
    probability times a scale to fp16 is off by 2^-11 (fp16 results keep what that leaves), the sums of the matrix instructions by 2^-15."""
    g = torch.Generator(device=DEV).manual_seed(n)
    q = (normal(1, 1, 2 * per, d).abs() + 0.5).to(dtype)
    scale = d**-0.5
    xk, xv = (torch.randn(1, 2, n, d, generator=g, device=DEV) for _ in range(2))
    xk *= 0.1
    for at in (0, n // 2, n - 1):
        k, v = xk.clone(), xv.clone()
        k[:, :, at] = -60 * math.log(2) / (scale * q.float().sum(-1).mean())
        v[:, :, at] *= 2.0**24
        out, lse, ref, ref_lse, size, _ = attend(q, k, v, kind, group, scale)
        # (the reach of the keys that count: scores of 0.1 and of the row far below, whose own probability does not matter)
        f = score_error(d, 1.0)
        part = f + 2.0**-15 + (2.0**-11 if dtype == torch.bfloat16 else 0.0)
        bound = part * size + torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        off = (out - ref).abs()
        assert (off <= bound).all(), f"row {at}: {(off / size).max().item():.3g} of the size"
        assert ((lse - ref_lse).abs() <= f + 2.0**-21 * ref_lse.abs()).all()


# Many items, so that a warp takes all keys of each.
BATCH, HEADS, KEYS = 230, 8, 512


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
@pytest.mark.parametrize("at", [0, 200, KEYS - 1])
def test_a_key_far_above_the_others_without_a_value(kind, group, dtype, at):
    """A sink: one key 2^18 above the others whose value is zero. What the others add is the result."""
    d, g = 64, torch.Generator(device=DEV).manual_seed(at)
    q = (normal(1, BATCH, 2 * HEADS, d).abs() + 0.5).to(dtype)
    scale = d**-0.5
    xk, xv = (torch.randn(BATCH, HEADS, KEYS, d, generator=g, device=DEV) for _ in range(2))
    xk *= 0.1
    xk[:, :, at] = 18 * math.log(2) / (scale * q.float().sum(-1).mean())
    xv[:, :, at] = 0
    out, _, ref, _, _, reach = attend(q, xk, xv * 4096, kind, group, scale)
    rows_close(out, ref, dtype, score_error(d, reach))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
@pytest.mark.parametrize("gap", [40, 46, 49, 50, 51, 52, 53, 54, 58])
def test_a_key_far_above_small_values(kind, group, gap):
    """Values of 2^-60 under a sink 2^40 to 2^58 above them, in the middle: products down to the end of fp32's normal numbers."""
    d, g = 64, torch.Generator(device=DEV).manual_seed(gap)
    q = torch.ones(BATCH, 2 * HEADS, d, device=DEV, dtype=torch.bfloat16)
    scale = d**-0.5
    xk, xv = (torch.randn(BATCH, HEADS, KEYS, d, generator=g, device=DEV) for _ in range(2))
    xk *= 0.1
    xk[:, :, 200] = gap * math.log(2) / (scale * d)
    xv[:, :, 200] = 0
    out, _, ref, _, _, reach = attend(q, xk, xv * 2.0**-60, kind, group, scale)
    rows_close(out, ref, torch.bfloat16, score_error(d, reach))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,group", [("int8", 64), ("e4m3", 64), ("int4", 64), ("int4", 32)])
@pytest.mark.parametrize("up", [False, True])
def test_scores_that_rise_as_values_fall(kind, group, dtype, up):
    """Probabilities rise (or fall) by 2^40 along the sequence, values do the opposite: every key weighs much the same."""
    d, g = 64, torch.Generator(device=DEV).manual_seed(7)
    q = (torch.ones(BATCH, 2 * HEADS, d, device=DEV) + normal(1, BATCH, 2 * HEADS, d, dtype=torch.float32) / 64).to(dtype)
    scale = d**-0.5
    xk, xv = (torch.randn(BATCH, HEADS, KEYS, d, generator=g, device=DEV) for _ in range(2))
    ramp = torch.linspace(-20, 20, KEYS, device=DEV).view(1, 1, -1, 1) * (1 if up else -1)
    xk = 0.1 * xk + ramp * math.log(2) / (scale * d)
    out, _, ref, _, _, reach = attend(q, xk, xv * torch.exp2(20 - ramp), kind, group, scale)
    rows_close(out, ref, dtype, score_error(d, reach))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(128, 64), (128, 32), (96, 32), (64, 32)])
def test_groups_of_columns_of_very_different_size(d, group, dtype):
    """4 bits: a group of columns 2^-20 of the others' size is as exact as they are."""
    b, h, n = 64, 4, 400
    g = torch.Generator(device=DEV).manual_seed(d)
    q, scale = normal(1, b, 4 * h, d, dtype=dtype), d**-0.5
    xk, xv = (torch.randn(b, h, n, d, generator=g, device=DEV) for _ in range(2))
    for small in range(d // group):
        columns = slice(small * group, (small + 1) * group)
        v = xv * 2.0**12
        v[..., columns] *= 2.0**-20
        out, _, ref, _, _, reach = attend(q, xk, v, "int4", group, scale)
        rows_close(out, ref, dtype, score_error(d, reach), columns)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20000, 70001])
@pytest.mark.parametrize("kind,d,group", [("int8", 128, 64), ("int4", 128, 64), ("int4", 96, 32), ("e4m3", 64, 64)])
def test_every_tile_of_a_long_sequence_counts(kind, d, group, n):
    """Values that average out: the result is far smaller than they are, and so is what it may be off by. bf16's rounding 2^-8, probabilities' 2^-11, the
    matrix instructions' at most 2^-8 (2^-14 of a code's step a key where a subnormal's exponent is taken for its size, all to one side: of the
    result's 4.6 steps / sqrt(n) in 4 bits 2^-8.2); 2^-7 in all. One tile of 32 rows that is not the right one is sqrt(64 / n), 0.03 and more, off."""
    import flash_sparse_attn as fsa

    q, cache = normal(5, 1, 8, d), make_cache(6, 1, n, 2, d, kind, group)
    out = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache)
    done()
    keys, vals = values(cache[0], cache[2])[0], values(cache[1], cache[3])[0]
    ref = reference(q, [keys], [vals], d**-0.5)[0]
    size = ref.norm(dim=-1)
    assert ((out.double().cpu() - ref).norm(dim=-1) <= 2.0**-7 * size).all()
    for tile in (0, n // 64, n // 32 - 1):  # what the bound has to see
        wrong = vals.clone()
        wrong[32 * tile:32 * tile + 32] = vals[:32].flip(0) if tile else vals[-32:]
        assert ((reference(q, [keys], [wrong], d**-0.5)[0] - ref).norm(dim=-1) > 2.0**-7 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d,group", [("int8", 128, 64), ("int4", 128, 32), ("e4m3", 64, 64)])
@pytest.mark.parametrize("chosen", [0, 9000])
def test_every_page_of_long_sequences_counts(kind, d, group, chosen):
    """The same for pages in any order, of sequences of several lengths, and for positions chosen among them: a page of values in another's place shows."""
    import flash_sparse_attn as fsa

    page, lens, g = 64, [20011, 4096, 11000], torch.Generator().manual_seed(3)
    slots = -(-max(lens) // page)
    table = torch.randperm(3 * slots + 2, generator=g)[:3 * slots].view(3, slots)
    q, cache = normal(5, 3, 8, d), make_cache(6, 3 * slots + 2, page, 2, d, kind, group)
    kw, pick = {}, [torch.arange(n) for n in lens]
    if chosen:
        at = torch.stack([torch.randperm(slots * page, generator=g)[:chosen].sort().values for _ in lens])
        kw["gather_kv_indices"], pick = at.to(torch.int32).to(DEV), [a[a < n] for a, n in zip(at, lens)]
    out = fsa.flash_dense_attn_with_quantized_kvcache_func(q, *cache, page_table=table.to(torch.int32).to(DEV),
                                                           seqused_k=torch.tensor(lens, dtype=torch.int32, device=DEV), **kw)
    done()
    pool = [values(cache[i], cache[2 + i]) for i in range(2)]
    keys, vals = ([x[table[i]].flatten(0, 1)[at] for i, at in enumerate(pick)] for x in pool)
    ref = reference(q, keys, vals, d**-0.5)[0]
    size = ref.norm(dim=-1)
    assert ((out.double().cpu() - ref).norm(dim=-1) <= 2.0**-7 * size).all()
    other = table.clone()
    other[:, [0, -1]] = table[:, [1, 2]]
    other[:, lens[1] // page - 1] = table[:, 5]
    wrong = [pool[1][other[i]].flatten(0, 1)[at] for i, at in enumerate(pick)]
    assert ((reference(q, keys, wrong, d**-0.5)[0] - ref).norm(dim=-1) > 2.0**-7 * size).all()
