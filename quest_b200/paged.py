"""Serving over a paged cache: the operators that a decoding loop needs around the W4A4 linears.

Keys and values lie in pools of pages ([num_pages, page_size, n_kv_head, head_dim]); a request's row of the page table lists its
pages in the order of its tokens, and the free pages are a stack on the device.  ``page_assign`` makes tables and slots of a step
from the requests' lengths, ``rope_paged_append`` rotates q and k and writes k and v into the pages, ``paged_attention`` attends
over them, ``verify_drafts`` checks drafted tokens and ``page_release`` takes pages back.  None of them reads a length on the
host, so a step can be captured in a CUDA graph and replayed while the requests grow.  ``quest_b200.serving`` puts them together.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib

_Strides6, _Strides10 = ctypes.c_longlong * 6, ctypes.c_longlong * 10


# These calls are short (a few microseconds on the device), so what Python does around them counts: types are compared by
# identity, devices by index, and entry points looked up once.
_i32, _bf16 = torch.int32, torch.bfloat16
_MOST_INT = 2 ** 31 - 1  # ctypes cuts a larger argument to 32 bits without a word
_entries: dict = {}


def _call(name: str, device: int, *args) -> None:
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if torch._C._cuda_getDevice() == device:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _lib.check(status, name)


class PageStep(NamedTuple):
    """What ``page_assign`` returns for a step; all tensors int32 except ``slots`` (int64)."""
    cu_new: torch.Tensor      # [batch + 1] first row of each request
    kv_lens: torch.Tensor     # [batch] tokens to attend over; 0: refused (or nothing there)
    lens: torch.Tensor        # [batch] tokens held after the step
    slots: torch.Tensor       # [num_tokens] where each row's key and value go, -1: nowhere
    positions: torch.Tensor   # [num_tokens] position of each row in its sequence
    free_count: torch.Tensor  # [1] free pages after the step


def page_assign(
        page_table: torch.Tensor,
        free_pages: torch.Tensor,
        free_count: torch.Tensor,
        cached_lens: torch.Tensor,
        new_lens: torch.Tensor,
        num_tokens: int,
        page_size: int,
) -> PageStep:
    """Pages, slots and positions of a step in which request b, ``cached_lens[b]`` tokens long, gets ``new_lens[b]`` more; their
    rows are packed one request after the other into ``num_tokens`` rows, those behind the last one unused.  New pages come from
    the end of the stack ``free_pages[:free_count]`` and are written into ``page_table`` [batch, width]; the other tensors stay
    as they are, so the caller goes on with the returned ``lens`` and ``free_count``.

    Requests are served in order.  One whose rows, table row or pages do not suffice is refused as a whole: it gets no page, its
    rows the slot -1 and its ``kv_lens`` is 0; where rows or pages have run out, so are the later ones that come behind them or need
    a page.  Negative lengths count as 0.  At most 8192 requests and 2^30 rows."""
    assert page_table.dtype is free_pages.dtype is free_count.dtype is cached_lens.dtype is new_lens.dtype is _i32
    assert (page_table.is_contiguous() and free_pages.is_contiguous() and free_count.is_contiguous() and cached_lens.is_contiguous()
            and new_lens.is_contiguous())
    assert page_table.dim() == 2 and free_pages.dim() == 1 and free_count.numel() == 1 and page_size > 0 and num_tokens >= 0
    assert num_tokens <= _MOST_INT and page_size <= _MOST_INT and free_pages.numel() <= _MOST_INT
    batch, width = page_table.shape
    assert cached_lens.shape == new_lens.shape == (batch,)
    dev = page_table.get_device()
    if dev < 0 or not dev == free_pages.get_device() == free_count.get_device() == cached_lens.get_device() == new_lens.get_device():
        _lib.require_cuda(page_table, free_pages, free_count, cached_lens, new_lens)
    cu, kv_lens, lens, positions, left = torch.split_with_sizes(page_table.new_empty(3 * batch + num_tokens + 2),
                                                                (batch + 1, batch, batch, num_tokens, 1))
    slots = page_table.new_empty(num_tokens, dtype=torch.int64)
    _call("page_assign_cuda", dev, page_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), cached_lens.data_ptr(),
          new_lens.data_ptr(), cu.data_ptr(), kv_lens.data_ptr(), lens.data_ptr(), slots.data_ptr(), positions.data_ptr(),
          left.data_ptr(), batch, width, free_pages.numel(), num_tokens, page_size)
    return PageStep(cu, kv_lens, lens, slots, positions, left)


def page_release(
        page_table: torch.Tensor,
        free_pages: torch.Tensor,
        free_count: torch.Tensor,
        lens: torch.Tensor,
        keep_lens: torch.Tensor,
        page_size: int,
) -> torch.Tensor:
    """Shortens request b from ``lens[b]`` to ``keep_lens[b]`` tokens (0: it has finished): the pages behind them go to the end of
    the stack ``free_pages[:free_count]``.  Returns the new count [1]; the page table is left as it is (what lies behind a
    request's length has no meaning).  ``free_pages`` must have room for every page of the pool (2^30 at most)."""
    assert page_table.dtype is free_pages.dtype is free_count.dtype is lens.dtype is keep_lens.dtype is _i32
    assert (page_table.is_contiguous() and free_pages.is_contiguous() and free_count.is_contiguous() and lens.is_contiguous()
            and keep_lens.is_contiguous())
    assert page_table.dim() == 2 and free_pages.dim() == 1 and free_count.numel() == 1 and page_size > 0
    assert page_size <= _MOST_INT and free_pages.numel() <= _MOST_INT
    batch, width = page_table.shape
    assert lens.shape == keep_lens.shape == (batch,)
    dev = page_table.get_device()
    if dev < 0 or not dev == free_pages.get_device() == free_count.get_device() == lens.get_device() == keep_lens.get_device():
        _lib.require_cuda(page_table, free_pages, free_count, lens, keep_lens)
    left = free_count.new_empty(1)
    _call("page_release_cuda", dev, page_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), lens.data_ptr(),
          keep_lens.data_ptr(), left.data_ptr(), batch, width, free_pages.numel(), page_size)
    return left


def rope_paged_append(
        qkv: torch.Tensor,
        table: torch.Tensor,
        positions: torch.Tensor,
        slots: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: torch.Tensor,
        n_head: int,
        q_out: torch.Tensor = None,
) -> torch.Tensor:
    """Rotates the queries and keys of qkv [rows, (n_head + 2 n_kv_head) head_dim] bf16 by row ``positions[r]`` of ``table``
    (length, head_dim/2, 2; fp32 or bf16; the same bits as ``rope_inplace``) and writes keys and values to ``slots[r]`` of the
    caches [num_pages, page_size, n_kv_head, head_dim].  Returns the queries [rows, n_head, head_dim].  Rows with a slot or a
    position outside (``page_assign`` gives -1 to rows that are not in use) are left out: nothing of them is written.  The slots
    of one call must differ.  For inference: nothing is recorded for autograd."""
    num_pages, page_size, n_kv_head, head_dim = k_cache.shape
    k_strides, v_strides = k_cache.stride(), v_cache.stride()
    assert k_cache.dtype is v_cache.dtype is _bf16 and v_cache.shape == k_cache.shape and k_strides[3] == v_strides[3] == 1
    assert qkv.dtype is _bf16 and qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.size(1) == (n_head + 2 * n_kv_head) * head_dim
    rows = qkv.size(0)
    assert (table.dtype is _bf16 or table.dtype is torch.float32) and table.is_contiguous() and table.shape[1:] == (head_dim // 2, 2)
    assert positions.dtype is _i32 and slots.dtype is torch.int64 and positions.is_contiguous() and slots.is_contiguous()
    assert positions.shape == slots.shape == (rows,)
    if q_out is None:
        q_out = qkv.new_empty((rows, n_head, head_dim))
    assert q_out.shape == (rows, n_head, head_dim) and q_out.dtype is _bf16 and q_out.is_contiguous()
    dev = qkv.get_device()
    if dev < 0 or not (dev == table.get_device() == positions.get_device() == slots.get_device() == k_cache.get_device() == v_cache.get_device()
                       == q_out.get_device()):
        _lib.require_cuda(qkv, table, positions, slots, k_cache, v_cache, q_out)
    strides = _Strides6(*k_strides[:3], *v_strides[:3])
    at = ctypes.addressof(strides)
    _call("rope_paged_append_cuda_bf16", dev, qkv.data_ptr(), qkv.stride(0) if rows > 1 else qkv.size(1), table.data_ptr(),
          table.dtype is _bf16, positions.data_ptr(), slots.data_ptr(), k_cache.data_ptr(), at, v_cache.data_ptr(), at + 24,
          q_out.data_ptr(), rows, n_head, n_kv_head, head_dim, table.size(0), num_pages, page_size)
    return q_out


@functools.lru_cache(maxsize=4096)
def _workspace(device: int, rows: int, group: int, head_dim: int) -> int:
    """Size of the workspace of an attention call in bf16 elements."""
    with torch.cuda.device(device):
        return _lib.load().paged_attention_workspace(rows, 1, group, 1, head_dim) // 2


def paged_attention(
        q: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: torch.Tensor,
        page_table: torch.Tensor,
        kv_lens: torch.Tensor,
        cu_new: torch.Tensor,
        scale: float = None,
        out: torch.Tensor = None,
) -> torch.Tensor:
    """softmax(scale q k^T) v of the new tokens of a step, causal, over the paged cache; ``scale`` is head_dim^-0.5 by default.

    Rows ``cu_new[b] .. cu_new[b + 1] - 1`` of q [rows, n_head, head_dim] bf16 are the last tokens of request b, whose
    ``kv_lens[b]`` tokens (the new ones among them) lie in the pages ``page_table[b]``: one row while decoding, a chunk of a
    prompt, drafted tokens, or a mixture over the batch.  Query head h reads key and value head h / (n_head / n_kv_head), at most
    128 of them the same.  Rows that see no key (kv_lens 0: refused by ``page_assign``) give zeros; rows outside every request are
    not written.  What the pages hold behind a request's tokens does not matter, nor what a row does not see (later tokens of its
    chunk, whatever they are).  head_dim 64 or 128, page_size a power of two from 16 to 1024, at most 2^20 requests; q and out may be views (strides in
    multiples of 8 elements), out without memory in common with the inputs.  For inference: nothing is recorded for autograd."""
    num_pages, page_size, n_kv_head, head_dim = k_cache.shape
    rows, n_head, columns = q.shape
    batch, width = page_table.shape
    q_strides, k_strides, v_strides = q.stride(), k_cache.stride(), v_cache.stride()
    assert q.dtype is k_cache.dtype is v_cache.dtype is _bf16 and v_cache.shape == k_cache.shape and columns == head_dim
    assert q_strides[2] == k_strides[3] == v_strides[3] == 1
    assert page_table.dtype is kv_lens.dtype is cu_new.dtype is _i32
    assert page_table.is_contiguous() and kv_lens.is_contiguous() and cu_new.is_contiguous()
    assert kv_lens.shape == (batch,) and cu_new.shape == (batch + 1,)
    if out is None:
        out = q.new_empty((rows, n_head, head_dim))
    out_strides = out.stride()
    assert out.shape == q.shape and out.dtype is _bf16 and out_strides[2] == 1
    dev = q.get_device()
    if dev < 0 or not (dev == k_cache.get_device() == v_cache.get_device() == page_table.get_device() == kv_lens.get_device()
                       == cu_new.get_device() == out.get_device()):
        _lib.require_cuda(q, k_cache, v_cache, page_table, kv_lens, cu_new, out)
    workspace = q.new_empty(_workspace(dev, rows, n_head // n_kv_head if n_kv_head else 0, head_dim))
    strides = _Strides10(*out_strides[:2], *q_strides[:2], *k_strides[:3], *v_strides[:3])
    at = ctypes.addressof(strides)
    _call("paged_attention_cuda_bf16", dev, out.data_ptr(), at, q.data_ptr(), at + 16, k_cache.data_ptr(), at + 32, v_cache.data_ptr(), at + 56,
          page_table.data_ptr(), kv_lens.data_ptr(), cu_new.data_ptr(), workspace.data_ptr(), head_dim ** -0.5 if scale is None else float(scale),
          rows, batch, width, n_head, n_kv_head, head_dim, num_pages, page_size)
    return out


def verify_drafts(
        target_probs: torch.Tensor,
        draft_tokens: torch.Tensor,
        cu_drafts: torch.Tensor,
        uniforms: torch.Tensor,
        max_drafts: int,
        draft_probs: torch.Tensor = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rejection sampling of drafted tokens: (tokens int64 [batch, max_drafts + 1], accepted int32 [batch]).

    Request b drafted ``draft_tokens[cu_drafts[b]:cu_drafts[b + 1]]`` (int64; possibly none).  Its rows of ``target_probs``
    [drafts + batch, vocab] (fp32 or bf16) and of ``uniforms`` [drafts + batch] (fp32, in [0, 1)) begin at ``cu_drafts[b] + b``
    and number one more than its drafts.  Draft i is kept while ``u_i * draft_probs[i, x_i] < target_probs[i, x_i]``; without
    ``draft_probs`` (same type, [drafts, vocab]) a draft has probability 1 in its own distribution.  The next token is drawn with
    the last uniform from max(target - draft, 0) of the first refused row, or from the row behind the last draft: the first whose
    running sum (in 64 bits) passes u times the total.  ``tokens`` holds the kept drafts, that token, and -1 behind it.  Drafts
    beyond ``max_drafts`` are not looked at.  Negative probabilities count as 0, and so does a NaN of the target's; a draft whose own
    probability is NaN is refused, and nothing is drawn where a draft's is NaN.  ``max_drafts`` and the drafts at most 2^30."""
    assert (target_probs.dtype is torch.float32 or target_probs.dtype is _bf16) and target_probs.dim() == 2 and target_probs.is_contiguous()
    assert draft_tokens.dtype is torch.int64 and draft_tokens.dim() == 1 and draft_tokens.is_contiguous()
    assert cu_drafts.dtype is _i32 and cu_drafts.dim() == 1 and cu_drafts.is_contiguous()
    n, batch, vocab = draft_tokens.numel(), cu_drafts.numel() - 1, target_probs.size(1)
    assert batch >= 0 and 0 <= max_drafts <= _MOST_INT and n <= _MOST_INT and target_probs.size(0) == n + batch
    assert uniforms.dtype is torch.float32 and uniforms.is_contiguous() and uniforms.shape == (n + batch,)
    assert draft_probs is None or (draft_probs.dtype is target_probs.dtype and draft_probs.shape == (n, vocab) and draft_probs.is_contiguous())
    dev = target_probs.get_device()
    if dev < 0 or not (dev == draft_tokens.get_device() == cu_drafts.get_device() == uniforms.get_device()
                       == (dev if draft_probs is None else draft_probs.get_device())):
        _lib.require_cuda(target_probs, draft_tokens, cu_drafts, uniforms, draft_probs)
    tokens = draft_tokens.new_empty((batch, max_drafts + 1))
    accepted = cu_drafts.new_empty(batch)
    # an empty draft_probs (no request has drafts) has no address and stands for nothing
    _call("verify_drafts_cuda", dev, target_probs.data_ptr(), _lib.ptr(draft_probs), target_probs.dtype is _bf16,
          draft_tokens.data_ptr(), cu_drafts.data_ptr(), uniforms.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), batch, n, vocab,
          max_drafts)
    return tokens, accepted
