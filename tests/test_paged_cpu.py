"""The serving operators without a GPU: refusals of the C entries and of the Python functions."""
from __future__ import annotations

import ctypes

import pytest
import torch

import quest_b200 as quest
from quest_b200 import _lib

OK, INVALID, UNSUPPORTED = 0, 1, 2


def aligned_buffer():
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    return buf, p + (-p) % 16


def test_page_entries_check_before_they_launch():
    lib = _lib.load()
    buf, p = aligned_buffer()
    assert lib.page_assign_cuda(*[p] * 11, -1, 4, 4, 4, 16, None) == INVALID
    assert lib.page_assign_cuda(*[p] * 11, 2, 4, 4, 4, 0, None) == INVALID
    assert lib.page_assign_cuda(*[p] * 10, None, 2, 4, 4, 4, 16, None) == INVALID
    assert lib.page_assign_cuda(None, *[p] * 10, 2, 4, 4, 4, 16, None) == INVALID
    assert lib.page_assign_cuda(*[p] * 11, 8193, 4, 4, 4, 16, None) == UNSUPPORTED
    assert lib.page_assign_cuda(*[p] * 11, 2, 1 << 27, 4, 4, 16, None) == UNSUPPORTED
    assert lib.page_release_cuda(*[p] * 6, 2, -1, 4, 16, None) == INVALID
    assert lib.page_release_cuda(*[p] * 3, None, p, p, 2, 4, 4, 16, None) == INVALID
    assert lib.page_release_cuda(*[p] * 6, 8193, 4, 4, 16, None) == UNSUPPORTED


def test_append_entry_checks_before_it_launches():
    lib = _lib.load()
    buf, p = aligned_buffer()
    good, odd = (ctypes.c_longlong * 3)(1024, 64, 64), (ctypes.c_longlong * 3)(1024, 60, 64)

    def call(qkv=p, ld=192, ks=good, q_out=p, rows=2, heads=1, d=64, page=16, pages=4):
        return lib.rope_paged_append_cuda_bf16(qkv, ld, p, 0, p, p, p, ks, p, good, q_out, rows, heads, 1, d, 8, pages, page, None)

    assert call(rows=0) == OK and call(pages=0) == OK
    assert call(rows=-1) == INVALID and call(qkv=None) == INVALID and call(ld=184) == INVALID and call(page=0) == INVALID and call(q_out=None) == INVALID
    assert call(ks=odd) == UNSUPPORTED and call(ld=196) == UNSUPPORTED and call(qkv=p + 2) == UNSUPPORTED and call(d=60) == UNSUPPORTED


def test_attention_entry_checks_before_it_launches():
    lib = _lib.load()
    buf, p = aligned_buffer()
    two, three = (ctypes.c_longlong * 2)(128, 64), (ctypes.c_longlong * 3)(1024, 64, 64)
    odd2, odd3 = (ctypes.c_longlong * 2)(128, 63), (ctypes.c_longlong * 3)(1028, 64, 64)

    def call(out=p, qs=two, ks=three, rows=2, batch=1, width=3, hq=2, hkv=1, d=64, pages=4, page=16, work=p, q=p):
        return lib.paged_attention_cuda_bf16(out, two, q, qs, p, ks, p, three, p, p, p, work, 0.1, rows, batch, width, hq, hkv, d, pages, page, None)

    assert call(rows=0) == OK and call(batch=0) == OK
    assert call(rows=-1) == INVALID and call(out=None) == INVALID and call(hkv=0) == INVALID and call(page=0) == INVALID
    for bad in (dict(d=96), dict(page=48), dict(page=8), dict(hq=3, hkv=2), dict(qs=odd2), dict(ks=odd3), dict(width=1 << 27), dict(q=p + 2)):
        assert call(**bad) == UNSUPPORTED, bad


def test_verify_entry_checks_before_it_launches():
    lib = _lib.load()
    buf, p = aligned_buffer()
    assert lib.verify_drafts_cuda(p, p, 0, p, p, p, p, p, 0, 0, 100, 4, None) == OK
    assert lib.verify_drafts_cuda(p, p, 0, p, p, p, p, p, 1, 0, 0, 4, None) == INVALID
    assert lib.verify_drafts_cuda(p, p, 0, p, p, p, p, p, 1, 2, 100, -1, None) == INVALID
    assert lib.verify_drafts_cuda(p, p, 0, None, p, p, p, p, 1, 2, 100, 4, None) == INVALID
    assert lib.verify_drafts_cuda(p, p, 0, p, p, p, p, p, 1, 2, (1 << 23) + 1, 4, None) == UNSUPPORTED


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _attend(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16),
             v_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16), page_table=_i32(2, 4), kv_lens=_i32(2), cu_new=_i32(3))
    a.update(kw)
    return quest.paged_attention(**a)


def _append(**kw):
    a = dict(qkv=torch.zeros(3, 8 * 64, dtype=torch.bfloat16), table=torch.zeros(9, 32, 2), positions=_i32(3), slots=torch.zeros(3, dtype=torch.int64),
             k_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16), v_cache=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16), n_head=4)
    a.update(kw)
    return quest.rope_paged_append(**a)


def _verify(**kw):
    a = dict(target_probs=torch.zeros(5, 50), draft_tokens=torch.zeros(3, dtype=torch.int64), cu_drafts=_i32(3), uniforms=torch.zeros(5), max_drafts=2)
    a.update(kw)
    return quest.verify_drafts(**a)


def _assign(**kw):
    a = dict(page_table=_i32(2, 4), free_pages=_i32(9), free_count=_i32(1), cached_lens=_i32(2), new_lens=_i32(2), num_tokens=3, page_size=16)
    a.update(kw)
    return quest.page_assign(**a)


def _release(**kw):
    a = dict(page_table=_i32(2, 4), free_pages=_i32(9), free_count=_i32(1), lens=_i32(2), keep_lens=_i32(2), page_size=16)
    a.update(kw)
    return quest.page_release(**a)


@pytest.mark.parametrize("op", [_attend, _append, _verify, _assign, _release])
def test_no_cpu_fallback(op):
    with pytest.raises(RuntimeError, match="CUDA"):
        op()


@pytest.mark.parametrize("op, bad", [
    (_attend, dict(q=torch.zeros(3, 4, 64))),
    (_attend, dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16))),
    (_attend, dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)[:, :, ::2])),
    (_attend, dict(kv_lens=_i32(3))),
    (_attend, dict(cu_new=_i32(2))),
    (_attend, dict(page_table=torch.zeros(2, 4, dtype=torch.int64))),
    (_attend, dict(out=torch.zeros(3, 4, 64))),
    (_attend, dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16))),
    (_attend, dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16))),
    (_append, dict(qkv=torch.zeros(3, 7 * 64, dtype=torch.bfloat16))),
    (_append, dict(table=torch.zeros(9, 64, 2))),
    (_append, dict(table=torch.zeros(9, 32, 2, dtype=torch.float16))),
    (_append, dict(slots=_i32(3))),
    (_append, dict(positions=_i32(4))),
    (_append, dict(q_out=torch.zeros(3, 4, 32, dtype=torch.bfloat16))),
    (_verify, dict(target_probs=torch.zeros(4, 50))),
    (_verify, dict(target_probs=torch.zeros(5, 50, dtype=torch.float16))),
    (_verify, dict(draft_probs=torch.zeros(3, 50, dtype=torch.bfloat16))),
    (_verify, dict(draft_probs=torch.zeros(2, 50))),
    (_verify, dict(uniforms=torch.zeros(4))),
    (_verify, dict(uniforms=torch.zeros(5, dtype=torch.float64))),
    (_verify, dict(draft_tokens=_i32(3))),
    (_assign, dict(new_lens=_i32(3))),
    (_assign, dict(cached_lens=torch.zeros(2, dtype=torch.int64))),
    (_assign, dict(free_count=_i32(2))),
    (_assign, dict(page_size=0)),
    (_assign, dict(num_tokens=-1)),
    (_release, dict(keep_lens=_i32(1))),
    (_release, dict(page_table=_i32(8))),
])
def test_arguments_are_checked(op, bad):
    with pytest.raises(AssertionError):
        op(**bad)


def test_attention_entry_refuses_scales_and_groups():
    lib = _lib.load()
    buf, p = aligned_buffer()
    two, three = (ctypes.c_longlong * 2)(64 * 256, 64), (ctypes.c_longlong * 3)(1024, 64, 64)

    def call(scale=0.1, hq=2, page=16, width=3):
        return lib.paged_attention_cuda_bf16(p, two, p, two, p, three, p, three, p, p, p, p, scale, 2, 1, width, hq, 1, 64, 4, page, None)

    assert call(scale=-1.0) == INVALID and call(scale=float("nan")) == INVALID
    assert call(hq=129) == UNSUPPORTED and call(page=2048) == UNSUPPORTED and call(width=(1 << 21) + 1) == UNSUPPORTED


def test_attention_entry_refuses_more_requests_than_it_can_walk_over_within_its_waits():
    lib = _lib.load()
    buf, p = aligned_buffer()
    two, three = (ctypes.c_longlong * 2)(64 * 256, 64), (ctypes.c_longlong * 3)(1024, 64, 64)
    assert lib.paged_attention_cuda_bf16(p, two, p, two, p, three, p, three, p, p, p, p, 0.1, 2, (1 << 20) + 1, 3, 2, 1, 64, 4, 16, None) == UNSUPPORTED


def test_pages_of_a_layer_refuse_where_a_gradient_is_asked_for():
    from quest_b200.serving import LayerPages
    k, v = (torch.zeros(5, 16, 4, 64, dtype=torch.bfloat16) for _ in range(2))
    step = quest.PageStep(_i32(2), _i32(1), _i32(1), torch.zeros(3, dtype=torch.int64), _i32(3), _i32(1))
    pages = LayerPages(k, v, _i32(1, 4), step)
    qkv, table = torch.zeros(3, 3 * 4 * 64, dtype=torch.bfloat16), torch.zeros(9, 32, 2)
    with pytest.raises(RuntimeError, match="gradient"):
        pages.attend(qkv.clone().requires_grad_(), table, 4)
    with pytest.raises(RuntimeError, match="gradient"), torch.autograd.forward_ad.dual_level():
        pages.attend(qkv, table, 4)
    with pytest.raises(RuntimeError, match="CUDA"):  # as far as the kernels
        pages.attend(qkv, table, 4)
    with pytest.raises(RuntimeError, match="CUDA"), torch.no_grad():
        pages.attend(qkv.clone().requires_grad_(), table, 4)


def test_entries_refuse_what_an_index_of_32_bits_cannot_walk_over():
    """Threads go through rows, pages and places in strides of a grid: near 2^31 the next index would be negative.  (Without a
    GPU a call that is not refused ends at its launch.)"""
    lib = _lib.load()
    buf, p = aligned_buffer()
    most, beyond = 2 ** 31 - 1, 2 ** 30 + 1
    for rows in (beyond, most):
        assert lib.page_assign_cuda(*[p] * 11, 2, 4, 4, rows, 16, None) == UNSUPPORTED
    for pool in (beyond, most):
        assert lib.page_release_cuda(*[p] * 6, 2, 4, pool, 16, None) == UNSUPPORTED
    for drafts, places in ((4, beyond), (4, most), (beyond, 4), (most, 4)):
        assert lib.verify_drafts_cuda(p, p, 0, p, p, p, p, p, 1, drafts, 100, places, None) == UNSUPPORTED
    strides = (ctypes.c_longlong * 3)(1024, 64, 64)
    for heads, kv_heads, d in ((1 << 27, 1, 8), (1, 1 << 30, 8), (most, most, most - 7)):
        assert lib.rope_paged_append_cuda_bf16(p, (1 << 62), p, 0, p, p, p, strides, p, strides, p, 1, heads, kv_heads, d, 8, 4, 16, None) == UNSUPPORTED


@pytest.mark.parametrize("op, bad", [(_assign, dict(num_tokens=2 ** 32 + 3)), (_assign, dict(page_size=2 ** 32 + 16)), (_release, dict(page_size=2 ** 32 + 16)),
                                     (_verify, dict(max_drafts=2 ** 32 + 2))])
def test_arguments_beyond_32_bits_are_not_cut(op, bad):
    with pytest.raises(AssertionError):
        op(**bad)
