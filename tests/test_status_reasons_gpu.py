"""The status word keeps the first reason: kernels that find it set leave without writing their results, and without a reason of
their own."""

import pytest
import torch

from test_rotary import launcher, normal, tables  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


def raised(status):
    import flash_sparse_attn as fsa

    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=f"device status {status} "):
        fsa.check_status()
    fsa.check_status()  # (cleared)


def no_room(rotary=True):
    """An append behind the end of its cache: status 3."""
    from flash_sparse_attn.utils.kvcache import append_kv, append_kv_rotary

    cos, sin = tables(64, 32)
    k, cache = normal(1, 1, 1, 2, 64), torch.zeros(1, 32, 2, 64, dtype=torch.bfloat16, device=DEV)
    if rotary:
        append_kv_rotary(None, k, k, cache, cache.clone(), torch.full((1,), 32, dtype=torch.int32, device=DEV), cos, sin)
    else:  # no page, and nothing to take one from
        table, used = torch.full((1, 1), -1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        append_kv(k, k, cache, cache.clone(), used, page_table=table)


def no_angles():
    """A position outside the tables: status 5."""
    import flash_sparse_attn as fsa

    cos, sin = tables(8, 32)
    fsa.apply_rotary_func(normal(1, 1, 9, 2, 64), None, cos, sin)


def shared_prefix(out=None, bad_page=None):
    import flash_sparse_attn as fsa

    q, k = normal(2, 40, 8, 64), normal(3, 40, 200, 2, 64)
    pool = normal(4, 20, 64, 2, 64)
    pages = torch.arange(20, dtype=torch.int32, device=DEV)
    if bad_page is not None:
        pages[7] = bad_page
    return fsa.flash_dense_attn_with_shared_prefix_func(q, k, k, pool, pool, prefix_page_table=pages, out=out)


def forward(out=None):
    import flash_sparse_attn as fsa

    q, k = normal(2, 2, 300, 4, 64), normal(3, 2, 300, 2, 64)
    return fsa.flash_dense_attn_func(q, k, k, is_causal=True, out=out)


@pytest.mark.parametrize("status,cause", [(3, no_room), (3, lambda: no_room(False)), (5, no_angles)], ids=["append rotary", "append", "rotary"])
@pytest.mark.parametrize("behind", [shared_prefix, forward])
def test_the_reason_outlives_the_kernels_behind_it(behind, status, cause):
    good = behind()
    cause()
    out = torch.full_like(good, 3.0)
    for _ in range(3):
        behind(out=out)
    raised(status)
    assert bool((out == 3.0).all())  # left as it was
    assert torch.equal(behind(out=out), good)
    raised_nothing()


def raised_nothing():
    import flash_sparse_attn as fsa

    torch.cuda.synchronize()
    fsa.check_status()


@pytest.mark.parametrize("status,cause", [(3, no_room), (5, no_angles)], ids=["append", "rotary"])
def test_the_reason_outlives_a_backward(status, cause):
    import flash_sparse_attn as fsa

    q, k = normal(2, 2, 300, 4, 64).requires_grad_(), normal(3, 2, 300, 2, 64)
    o = fsa.flash_dense_attn_func(q, k, k, is_causal=True)
    cause()
    o.backward(torch.ones_like(o))
    raised(status)


def test_the_first_reason_stands():
    no_room(), no_angles(), no_room(False)
    raised(3)
    no_angles(), no_room(), no_room(False)
    raised(5)
    no_room(False), no_angles()
    raised(3)
    shared_prefix(bad_page=1 << 20), no_angles(), shared_prefix()
    raised(3)
    no_angles(), shared_prefix(bad_page=-1)
    raised(5)


def test_a_page_outside_the_pool_is_reported_as_that():
    for _ in range(20):
        shared_prefix(bad_page=20)
        raised(3)


def test_the_word_is_set_and_cleared_while_calls_are_under_way():
    """A call of two kernels may find the word set in the first and cleared in the second, which then meets what the first has not
    written: it must not take that for places to read from."""
    import flash_sparse_attn as fsa
    from flash_sparse_attn import _lib

    word = _lib.status_word(torch.device(DEV, torch.cuda.current_device()))
    good = shared_prefix()
    torch.cuda.synchronize()
    q, k = normal(2, 40, 8, 64), normal(3, 40, 200, 2, 64)
    pool, pages = normal(4, 20, 64, 2, 64), torch.arange(20, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    seen = 0
    for i in range(200):
        with torch.cuda.stream(side):
            torch.full((1 << 20,), -1.0, device=DEV)  # what a workspace is then made of: not places
            for _ in range(4):
                fsa.flash_dense_attn_with_shared_prefix_func(q, k, k, pool, pool, prefix_page_table=pages)
        word.fill_(7)
        for _ in range(i % 4):
            word.zero_()
            word.fill_(7)
        try:
            fsa.check_status()
        except RuntimeError as e:
            seen += "device status 7 " in str(e)
    torch.cuda.synchronize()
    word.zero_()
    assert seen > 0
    assert torch.equal(shared_prefix(), good)
    raised_nothing()
