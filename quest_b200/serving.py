"""Decoding with the Llama-style decoder of ``prefill.py`` over a paged cache.

``PagedCache`` owns the pages of every layer and the bookkeeping on the device; ``extend`` runs the new tokens of all requests
(prompts, chunks of prompts, single tokens, drafts, in any mixture) through the model in one packed batch; ``generate`` is the
greedy loop and ``verify`` one step of speculative decoding.  The reference stops at one forward pass without logits
(gemm-quest/benchmarks/bench_e2e.py:98-121); its decoder has no cache.
"""
from __future__ import annotations

import torch

import quest_b200 as quest
from .paged import PageStep
from .prefill import Decoder, DecoderConfig, kernels_may_replace


class LayerPages:
    """One layer's pages during one step: what its attention needs in place of dense keys and values."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, step: PageStep):
        self.k, self.v, self.page_table, self.step = k, v, page_table, step

    def attend(self, qkv: torch.Tensor, table: torch.Tensor, n_head: int) -> torch.Tensor:
        """qkv [rows, 3 n_head head_dim], not rotated yet -> attention [rows, n_head, head_dim]; keys and values go to the pages.
        Rows that belong to no request come out as zeros.  For inference: refused where a gradient is asked for."""
        if not kernels_may_replace(qkv, table, self.k, self.v):
            raise RuntimeError("attention over pages leaves no graph for a gradient: run the model under torch.no_grad() or torch.inference_mode()")
        head_dim = self.k.size(3)
        rows = qkv.size(0)
        q = quest.rope_paged_append(qkv, table, self.step.positions, self.step.slots, self.k, self.v, n_head)
        out = torch.zeros(rows, n_head, head_dim, dtype=qkv.dtype, device=qkv.device)
        return quest.paged_attention(q, self.k, self.v, self.page_table, self.step.kv_lens, self.step.cu_new, out=out)


class PagedCache:
    """Pages of all layers of a model for up to ``max_requests`` requests of up to ``max_length`` tokens; ``num_pages`` pages of
    ``page_size`` tokens are shared by them.  ``lens`` [max_requests] are the tokens held, on the device."""

    def __init__(self, cfg: DecoderConfig, num_pages: int, max_requests: int, max_length: int = None, page_size: int = 64, device="cuda"):
        head_dim = cfg.n_embd // cfg.n_head
        max_length = cfg.sequence_length if max_length is None else max_length
        assert page_size > 0 and 0 < max_length <= cfg.sequence_length, "up to the end of the rotary table"
        self.page_size, self.num_pages, self.max_length = page_size, num_pages, max_length
        self.k, self.v = ([torch.zeros(num_pages, page_size, cfg.n_head, head_dim, dtype=torch.bfloat16, device=device)
                           for _ in range(cfg.n_layer)] for _ in range(2))
        self.page_table = torch.zeros(max_requests, -(-max_length // page_size), dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=device)

    def assign(self, new_lens: torch.Tensor, num_tokens: int) -> PageStep:
        """Room for ``new_lens[b]`` more tokens of every request; requests without room are refused (``page_assign``)."""
        lens, room = self.lens, self.page_table.size(1) * self.page_size
        if room > self.max_length:  # the table's last page goes beyond max_length: who would, too, is refused as one who has no page left
            beyond = new_lens > self.max_length - lens
            lens = torch.where(beyond, room, lens)
        step = quest.page_assign(self.page_table, self.free_pages, self.free_count, lens, new_lens, num_tokens, self.page_size)
        if room > self.max_length:
            step = step._replace(lens=torch.where(beyond, self.lens, step.lens))
        self.lens.copy_(step.lens)
        self.free_count.copy_(step.free_count)
        return step

    def shorten(self, keep_lens: torch.Tensor) -> None:
        """Request b keeps its first ``keep_lens[b]`` tokens (0: it has finished and its place can be used again)."""
        keep = torch.minimum(keep_lens, self.lens).clamp(min=0)
        self.free_count.copy_(quest.page_release(self.page_table, self.free_pages, self.free_count, self.lens, keep, self.page_size))
        self.lens.copy_(keep)

    def layers(self, step: PageStep) -> list[LayerPages]:
        return [LayerPages(k, v, self.page_table, step) for k, v in zip(self.k, self.v)]


@torch.inference_mode()
def extend(model: Decoder, cache: PagedCache, tokens: torch.Tensor, new_lens: torch.Tensor) -> tuple[torch.Tensor, PageStep]:
    """Runs ``tokens`` [rows], the new tokens of the requests packed one after the other (``new_lens`` [max_requests] int32 of
    them; rows behind the last are padding), through the model.  Returns (hidden states [rows, n_embd], step).  Nothing is
    read on the host: a step of fixed size can be captured in a graph and replayed."""
    rows = tokens.reshape(1, -1)
    step = cache.assign(new_lens, rows.size(1))
    return model(rows, cache.layers(step))[0], step


def last_rows(step: PageStep) -> torch.Tensor:
    """Row of each request's last new token (0 where it has none)."""
    return (step.cu_new[1:] - 1).clamp(min=0).long()


@torch.inference_mode()
def generate(model: Decoder, cache: PagedCache, prompts: list[torch.Tensor], max_new: int) -> torch.Tensor:
    """Greedy continuation of the prompts (1-D token ids, at most ``max_requests``): [len(prompts), max_new].  The requests take the
    first places of the cache, which must be free, and give their pages back at the end."""
    slots, n = cache.lens.numel(), len(prompts)
    device = cache.lens.device
    if n > slots or any(p.numel() == 0 for p in prompts):
        raise ValueError("more prompts than places, or an empty prompt")
    if bool((cache.lens[:n] != 0).any()):
        raise ValueError("places of the cache are in use")
    held = [p.numel() + max(max_new - 1, 0) for p in prompts]  # the last new token is not kept
    if max(held, default=0) > cache.max_length:
        raise ValueError(f"a prompt and its continuation are longer than the cache's length of {cache.max_length} tokens")
    if sum(-(-h // cache.page_size) for h in held) > int(cache.free_count):
        raise ValueError("the cache has too few free pages for these prompts and their continuation")
    if n == 0:
        return torch.empty(0, max_new, dtype=torch.long, device=device)
    new = torch.zeros(slots, dtype=torch.int32, device=device)
    new[:n] = torch.tensor([p.numel() for p in prompts], dtype=torch.int32, device=device)
    hidden, step = extend(model, cache, torch.cat([p.to(device) for p in prompts]), new)
    new[:n] = 1
    result = []
    for i in range(max_new):
        token = model.lm_head(hidden[last_rows(step)[:n]]).argmax(dim=-1)
        result.append(token)
        if i + 1 < max_new:
            hidden, step = extend(model, cache, token, new)
    keep = cache.lens.clone()
    keep[:n] = 0
    cache.shorten(keep)
    return torch.stack(result, dim=1) if result else torch.empty(n, 0, dtype=torch.long, device=device)


@torch.inference_mode()
def verify(model: Decoder, cache: PagedCache, tokens: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor,
           draft_probs: torch.Tensor = None, active: torch.Tensor = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One step of speculative decoding for all places of the cache: ``tokens`` [R], the last token of each request, which is not
    in the cache yet, and ``drafts`` [R, K] drafted behind it run through the model in one pass, drafts that the target refuses are taken
    out of the cache again.  ``uniforms`` [R, K + 1] fp32 in [0, 1); ``draft_probs`` [R, K, vocab] fp32.  Returns (new tokens
    [R, K + 1], -1 behind the last one; drafts kept [R]); the last new token is the next call's ``tokens``.  Places that are not
    ``active`` ([R] bool; all are by default) stay as they are, whatever their tokens are; they, and requests for which there are not
    enough pages, get -1 throughout and 0.  Arguments are checked before the cache changes."""
    device = cache.lens.device
    if drafts.dim() != 2 or drafts.size(0) != cache.lens.numel() or drafts.dtype != torch.int64 or tokens.shape != drafts.shape[:1]:
        raise ValueError("tokens [R] and drafts [R, K] int64, R the places of the cache")
    requests, count = drafts.shape
    rows, vocab = requests * (count + 1), model.lm_head.out_features
    if uniforms.numel() != rows or uniforms.dtype != torch.float32:
        raise ValueError("uniforms [R, K + 1] fp32")
    if draft_probs is not None and (draft_probs.numel() != requests * count * vocab or draft_probs.dtype != torch.float32):
        raise ValueError("draft_probs [R, K, vocab] fp32")
    if active is not None and (active.shape != (requests,) or active.dtype != torch.bool):
        raise ValueError("active [R] bool")
    if any(t is not None and t.device != device for t in (tokens, drafts, uniforms, draft_probs, active)):
        raise ValueError(f"all tensors on the device of the cache, {device}")
    before = cache.lens.clone()
    new = torch.full((requests,), count + 1, dtype=torch.int32, device=device)
    packed = torch.cat([tokens[:, None], drafts], dim=1).view(-1)
    if active is not None:  # the active places' tokens move together; place b's begin at its row of the packed batch
        new = torch.where(active, new, 0)
        ends = new.cumsum(0)
        at = ((ends - new)[:, None] + torch.arange(count + 1, device=device)).view(-1)
        idle = ~active.repeat_interleave(count + 1, output_size=rows)
        packed = packed.new_zeros(rows + 1).scatter_(0, at.masked_fill(idle, rows), packed)[:rows]
    hidden, step = extend(model, cache, packed, new)
    if active is not None:
        hidden = hidden[at.clamp(max=rows - 1)]
    probs = torch.softmax(model.lm_head(hidden).float(), dim=-1)
    cu = torch.arange(requests + 1, dtype=torch.int32, device=device) * count
    result, kept = quest.verify_drafts(probs, drafts.reshape(-1), cu, uniforms.reshape(-1), count,
                                       draft_probs=None if draft_probs is None else draft_probs.reshape(requests * count, vocab))
    served = step.kv_lens > 0
    if active is not None:
        served &= active
    cache.shorten(torch.where(served, before + 1 + kept, before))
    return torch.where(served[:, None], result, -1), torch.where(served, kept, 0)
