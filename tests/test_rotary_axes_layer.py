"""The attention layer with positions on several axes: the step goes through the operator, results and gradients are the formula's."""

import pytest
import torch

DEV = "cuda"


def turn(x, cos, sin):
    """The formula in fp32, rounded once, as plain operations with autograd's own gradient."""
    c, s = cos[..., None, :], sin[..., None, :]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def owners(sections, dealt):
    """The axis of each pair."""
    if dealt:
        return [i % 3 if i // 3 < sections[i % 3] else 0 for i in range(32)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


@pytest.mark.gpu
@pytest.mark.parametrize("sections, dealt", [((8, 12, 12), False), ((12, 10, 10), True)])
def test_layer_turns_by_several_axes(sections, dealt):
    from flash_sparse_attn.modules.flash_sparse_attention import FlashSparseAttention, FlashSparseAttentionConfig
    from flash_sparse_attn.ops.triton.interface import flash_gated_attn_func

    torch.manual_seed(0)
    layer = FlashSparseAttention(FlashSparseAttentionConfig(256, 8, 2, 64, softmax_threshold=-128.0, gate_threshold=-128.0)).to(DEV, torch.bfloat16)
    x = torch.randn(2, 150, 256, device=DEV, dtype=torch.bfloat16)
    angles = torch.arange(200.0, device=DEV)[:, None] * 10000.0 ** (-torch.arange(32.0, device=DEV) / 32)
    cos, sin = angles.cos(), angles.sin()
    ids = torch.randint(0, 200, (3, 2, 150), generator=torch.Generator().manual_seed(1)).to(DEV)
    pick = lambda table: torch.stack([table[ids[a], i] for i, a in enumerate(owners(sections, dealt))], -1)  # noqa: E731  [B, S, 32]

    inp = x.clone().requires_grad_()
    out, (keys, values) = layer(inp, rotary=(cos, sin), position_ids=ids, rotary_sections=sections, rotary_axes_dealt=dealt)
    g = torch.randn_like(out)
    got = torch.autograd.grad(out, [inp, *layer.parameters()], g)
    ref_in = x.clone().requires_grad_()
    heads = lambda w, n: torch.nn.functional.linear(ref_in, w.weight).view(2, 150, n, 64)  # noqa: E731
    q, k = turn(heads(layer.q_proj, 8), pick(cos), pick(sin)), turn(heads(layer.k_proj, 2), pick(cos), pick(sin))
    v = heads(layer.v_proj, 2)
    alpha, delta = (torch.nn.functional.linear(ref_in, w.weight) for w in (layer.a_proj, layer.d_proj))
    ref = layer.o_proj(flash_gated_attn_func(q, k, v, alpha, delta, is_causal=True, softmax_scale=layer.scaling,
                                             softmax_threshold=-128.0, gate_threshold=-128.0).reshape(2, 150, -1))
    want = torch.autograd.grad(ref, [ref_in, *layer.parameters()], g)
    # a rounding of the rotation may fall the other way (half a step, 2^-8, of single elements of q and k), which the 16-bit
    # probabilities and projections behind it (2^-8 each) pass on: 2^-6 of the largest element covers four such
    for a, b in ((keys, k), (values, v), (out, ref), *zip(got, want)):
        assert (a.float() - b.float()).abs().max() <= 2.0**-6 * b.float().abs().max()
    one_axis, _ = layer(x, rotary=(cos, sin), position_ids=ids[0])
    assert not torch.equal(one_axis, out)


def test_layer_calls_the_operator(monkeypatch):
    from flash_sparse_attn.modules import flash_sparse_attention as module

    seen = {}

    def operator(q, k, cos, sin, position_ids, sections, **kw):
        seen.update(kw, tables=(cos, sin), ids=position_ids, sections=sections)
        return q + 1, k + 2

    monkeypatch.setattr(module, "apply_rotary_axes_func", operator)
    monkeypatch.setattr(module, "apply_rotary_func", lambda *a, **kw: pytest.fail("one axis"))
    monkeypatch.setattr(module, "flash_gated_attn_func", lambda q, k, v, *a, **kw: seen.update(q=q, k=k) or q)
    layer = module.FlashSparseAttention(module.FlashSparseAttentionConfig(64, 4, 2, 16))
    _, (keys, _) = layer(torch.zeros(1, 3, 64), rotary=("cos", "sin"), position_ids="ids", rotary_sections=(4, 4), rotary_axes_dealt=True)
    assert seen["tables"] == ("cos", "sin") and seen["ids"] == "ids" and seen["sections"] == (4, 4)
    assert seen["axes_dealt"] is True and seen["interleaved"] is False
    assert (seen["q"] == 1).all() and (keys == 2).all()


def test_layer_refuses_axes_that_turn_nothing():
    from flash_sparse_attn.modules.flash_sparse_attention import FlashSparseAttention, FlashSparseAttentionConfig

    layer, x = FlashSparseAttention(FlashSparseAttentionConfig(64, 4, 2, 16)), torch.zeros(1, 3, 64)
    for kw in (dict(rotary_sections=(4, 4)), dict(rotary_sections=(4, 4), position_ids=torch.zeros(2, 1, 3, dtype=torch.int32)),
               dict(rotary=(torch.ones(4, 8), torch.ones(4, 8)), rotary_axes_dealt=True), dict(rotary_axes_dealt=True)):
        with pytest.raises(AssertionError, match="belong"):
            layer(x, **kw)


def test_sections_are_whole_numbers_whatever_was_called_before():
    from flash_sparse_attn.ops.triton.rotary_axes import axis_bits

    assert axis_bits((1, 31), 32, False) == axis_bits((1, 31), 32, False)
    for bad in ((1.0, 31), (True, 31), (1, 31.0)):
        with pytest.raises(AssertionError):
            axis_bits(bad, 32, False)
