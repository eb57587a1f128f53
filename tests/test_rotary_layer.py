"""The attention layer with rotary positions: the step goes through the operator, results and gradients are those of the formula."""

import pytest
import torch

from test_rotary import tables

DEV = "cuda"


def turn(x, cos, sin):
    """The formula in fp32, rounded once, as plain operations with autograd's own gradient."""
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


@pytest.mark.gpu
def test_layer_turns_queries_and_keys():
    from flash_sparse_attn.modules.flash_sparse_attention import FlashSparseAttention, FlashSparseAttentionConfig
    from flash_sparse_attn.ops.triton.interface import flash_gated_attn_func

    torch.manual_seed(0)
    layer = FlashSparseAttention(FlashSparseAttentionConfig(256, 8, 2, 64, softmax_threshold=-128.0, gate_threshold=-128.0)).to(DEV, torch.bfloat16)
    x = torch.randn(2, 200, 256, device=DEV, dtype=torch.bfloat16)
    cos, sin = tables(300, 32)
    ids = torch.stack([torch.arange(200) + 90, torch.arange(200)]).to(DEV)
    for position_ids in (None, ids):
        inp = x.clone().requires_grad_()
        out, (keys, values) = layer(inp, rotary=(cos, sin), position_ids=position_ids)
        g = torch.randn_like(out)
        got = torch.autograd.grad(out, [inp, *layer.parameters()], g)
        ref_in = x.clone().requires_grad_()
        heads = lambda w, n: torch.nn.functional.linear(ref_in, w.weight).view(2, 200, n, 64)  # noqa: E731
        at = ids if position_ids is not None else torch.arange(200, device=DEV).expand(2, -1)
        q, k = (torch.stack([turn(t[i], cos[at[i]], sin[at[i]]) for i in range(2)]) for t in (heads(layer.q_proj, 8), heads(layer.k_proj, 2)))
        v = heads(layer.v_proj, 2)
        alpha, delta = (torch.nn.functional.linear(ref_in, w.weight) for w in (layer.a_proj, layer.d_proj))
        ref = layer.o_proj(flash_gated_attn_func(q, k, v, alpha, delta, is_causal=True, softmax_scale=layer.scaling,
                                                 softmax_threshold=-128.0, gate_threshold=-128.0).reshape(2, 200, -1))
        want = torch.autograd.grad(ref, [ref_in, *layer.parameters()], g)
        # a rounding of the rotation may fall the other way (half a step, 2^-8, of single elements of q and k), which the 16-bit
        # probabilities and projections behind it (2^-8 each) pass on: 2^-6 of the largest element covers four such
        for a, b in ((keys, k), (values, v), (out, ref), *zip(got, want)):
            assert (a.float() - b.float()).abs().max() <= 2.0**-6 * b.float().abs().max()
        assert not torch.equal(keys, heads(layer.k_proj, 2))
    plain, _ = layer(x)
    assert not torch.equal(plain, out)


def test_layer_calls_the_operator(monkeypatch):
    from flash_sparse_attn.modules import flash_sparse_attention as module

    seen = {}

    def operator(q, k, cos, sin, **kw):
        seen.update(kw, tables=(cos, sin), shapes=(q.shape, k.shape))
        return q + 1, k + 2

    monkeypatch.setattr(module, "apply_rotary_func", operator)
    monkeypatch.setattr(module, "flash_gated_attn_func", lambda q, k, v, *a, **kw: seen.update(q=q, k=k) or q)
    layer = module.FlashSparseAttention(module.FlashSparseAttentionConfig(64, 4, 2, 16))
    x = torch.zeros(1, 3, 64)
    _, (keys, _) = layer(x, rotary=("cos", "sin"), position_ids="ids", rotary_interleaved=True)
    assert seen["tables"] == ("cos", "sin") and seen["position_ids"] == "ids" and seen["interleaved"] is True
    assert seen["shapes"] == ((1, 3, 4, 16), (1, 3, 2, 16)) and (seen["q"] == 1).all() and (keys == 2).all()
    seen.clear()
    layer(x)
    assert "tables" not in seen and not seen["q"].any()


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_a_compiled_step_is_the_same():
    """The compiler cuts its graph at the three operators of a step."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn.utils.kvcache import append_kv_rotary

    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(3, 1, h, 64, generator=g).to(torch.bfloat16).to(DEV) for h in (4, 2, 2))
    pk, pv = (torch.randn(40, 2, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    cos, sin = (torch.randn(60, 32, generator=g).to(DEV) for _ in range(2))
    weight = torch.randn(3, 1, 4, 64, generator=g).to(torch.bfloat16).to(DEV)

    def step(q, k, v, kc, vc, used):
        turned = append_kv_rotary(q + 1, k, v, kc, vc, used, cos, sin, seqlen_offsets=40)
        return fsa.flash_dense_attn_with_shared_prefix_func(turned[:, 0], kc, vc, pk, pv, seqused_k=used) * 2

    def loss(q):
        return (fsa.apply_rotary_func(q + 1, None, cos, sin) * weight).sum()

    results = []
    for run in (step, torch.compile(step, backend="eager")):
        kc, vc = (torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        used = torch.tensor([0, 3, 7], dtype=torch.int32, device=DEV)
        results.append((run(q, k, v, kc, vc, used), kc, vc, used))
    for run in (loss, torch.compile(loss, backend="eager")):
        x = q.clone().requires_grad_()
        results.append((torch.autograd.grad(run(x), x)[0],))
    torch.cuda.synchronize()
    fsa.check_status()
    for a, b in (results[:2], results[2:]):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
