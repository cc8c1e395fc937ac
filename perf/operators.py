"""The operators of serving over a paged cache: the calls whose speed counts, in their plain form and through the package.

Kinds:
  assign   ``page_assign``: page tables, slots and positions of a step from the requests' lengths
  release  ``page_release``: pages of finished requests or refused drafts back to the free list
  append   ``rope_paged_append``: rotary embedding of q and k, k and v into the pages
  attend   ``paged_attention``: new tokens (one or a chunk per request) over the pages
  verify   ``verify_drafts``: drafted tokens against the target's probabilities, the next token sampled
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # a decoding step of 64 sequences: one new token each, a page now and then
        {"name": "assign_64", "kind": "assign", "batch": 64, "kv": 4096, "new": 1, "page": 16, "pad": 0},
        # prompts of 512 requests, of different lengths and some of them empty, packed into one step with rows to spare
        {"name": "assign_512", "kind": "assign", "batch": 512, "kv": 2048, "new": 128, "page": 32, "pad": 777},
        # drafts refused in 64 sequences: a few tokens each are taken back
        {"name": "release_64", "kind": "release", "batch": 64, "kv": 4096, "drop": 8, "page": 16},
        # half of 1000 long sequences have finished
        {"name": "release_1000", "kind": "release", "batch": 1000, "kv": 8192, "drop": 0, "page": 64},
        # a decoding step of 33 sequences through the 800M decoder (16 heads)
        {"name": "append_33", "kind": "append", "batch": 33, "new": 1, "hq": 16, "hkv": 16, "d": 128, "page": 64, "pad": 0, "table": "bf16"},
        # 16 prompts of 1024 tokens, the 70B layer's shared heads (projection of 10240 columns)
        {"name": "append_16384", "kind": "append", "batch": 16, "new": 1024, "hq": 64, "hkv": 8, "d": 128, "page": 64, "pad": 0, "table": "fp32"},
        # one sequence decoding behind a prompt of 1000 tokens in the 800M decoder: latency
        {"name": "decode_1", "kind": "attend", "mode": "decode", "batch": 1, "kv": 1001, "new": 1, "hq": 16, "hkv": 16, "d": 128, "page": 64, "pad": 0},
        # 64 sequences of very different lengths decoding with shared heads: the stream over the cache
        {"name": "decode_64", "kind": "attend", "mode": "decode", "batch": 64, "kv": 16384, "new": 1, "hq": 64, "hkv": 8, "d": 128, "page": 16, "pad": 0},
        # the prefill the benchmark reports: 16 prompts of 1024 tokens, 16 heads
        {"name": "prefill_16x1024", "kind": "attend", "mode": "prefill", "batch": 16, "kv": 1024, "new": 1024, "hq": 16, "hkv": 16, "d": 128, "page": 64, "pad": 0},
        # a chunk of 4096 tokens of one long prompt among 15 decoding sequences
        {"name": "chunk_4096", "kind": "attend", "mode": "mixed", "batch": 16, "kv": 32768, "new": 4096, "hq": 64, "hkv": 8, "d": 128, "page": 128, "pad": 0},
        # four drafted tokens in each of 7 sequences, the vocabulary of the 800M decoder
        {"name": "verify_7", "kind": "verify", "batch": 7, "drafts": 4, "vocab": 32000, "draft_probs": True, "dtype": "fp32"},
        # a serving batch with up to eight drafts each and a large vocabulary
        {"name": "verify_200", "kind": "verify", "batch": 200, "drafts": 8, "vocab": 131072, "draft_probs": True, "dtype": "bf16"},
    ]


_HEADS = [(16, 16), (32, 32), (64, 8), (32, 8), (28, 4), (13, 13), (12, 2), (8, 1), (5, 5)]
_MOST_FLOPS = 4 * 128 * 64 * 4096 * 30720  # chunk_4096
_MOST_KV = 64 * 16384 * 8 * 128            # elements of K over the pages: decode_64 if all of its sequences were long


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choices(["attend", "append", "assign", "release", "verify"], [6, 2, 2, 1, 2])[0]
    page = rng.choice([16, 32, 64, 128])
    if kind == "assign":
        new = rng.choice([1, 1, _log_int(rng, 2, 256)])
        return {"kind": kind, "batch": _log_int(rng, 1, 1024 if new == 1 else 256), "kv": _log_int(rng, 64, 16384), "new": new, "page": page,
                "pad": rng.choice([0, rng.randint(1, 1000)])}
    if kind == "release":
        return {"kind": kind, "batch": _log_int(rng, 1, 1024), "kv": _log_int(rng, 64, 8192), "drop": rng.choice([0, rng.randint(1, 16)]), "page": page}
    if kind == "verify":
        return {"kind": kind, "batch": _log_int(rng, 1, 128), "drafts": rng.randint(1, 8), "vocab": _log_int(rng, 1000, 131072),
                "draft_probs": rng.random() < 0.7, "dtype": rng.choice(["fp32", "bf16"])}
    hq, hkv = rng.choice(_HEADS)
    d = rng.choice([64, 128])
    pad = rng.choice([0, 0, rng.randint(1, 40)])
    if kind == "append":
        new = rng.choice([1, _log_int(rng, 2, 1024)])
        most = min(256, 16384 * 80 * 128 // (new * (hq + 2 * hkv) * d))
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, most)), "new": new, "hq": hq, "hkv": hkv, "d": d, "page": page, "pad": pad,
                "table": rng.choice(["fp32", "bf16"])}
    mode = rng.choice(["decode", "decode", "prefill", "mixed"])
    kv = _log_int(rng, 17, 32768 if mode != "prefill" else 8192)
    batch = max(1, min(_log_int(rng, 1, 128), _MOST_KV // (kv * hkv * d)))
    new = rng.randint(1, 5) if mode == "decode" else kv if mode == "prefill" else _log_int(rng, 1, min(kv, 4096))
    if mode == "prefill":
        batch = max(1, min(batch, _MOST_FLOPS // (2 * d * hq * kv * kv), 32768 // kv))
    return {"kind": kind, "mode": mode, "batch": batch, "kv": kv, "new": min(new, kv), "hq": hq, "hkv": hkv, "d": d, "page": page, "pad": pad}


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens in the cache before the step, new tokens) of every request.  They follow from the case alone."""
    rng = random.Random("lengths %s" % sorted((k, v) for k, v in case.items() if k != "name"))
    kind, batch = case["kind"], case["batch"]
    if kind == "append":
        new = [case["new"] if i == 0 or case["new"] == 1 else rng.randint(1, case["new"]) if batch % 16 else case["new"] for i in range(batch)]
        return [rng.randint(0, 900) for _ in range(batch)], new
    if kind == "assign":
        new = [1 if case["new"] == 1 else rng.choice([0, case["new"], rng.randint(1, case["new"])]) for _ in range(batch)]
        return [0 if case["new"] > 1 and rng.random() < 0.5 else _log_int(rng, 1, case["kv"]) for _ in range(batch)], new
    if kind == "release":
        return [_log_int(rng, 1, case["kv"]) for _ in range(batch)], [0] * batch
    if case["mode"] == "prefill":  # prompts of one length, or of many where the batch is not a power of two
        new = [case["kv"] if i == 0 or batch & (batch - 1) == 0 else rng.randint(1, case["kv"]) for i in range(batch)]
        return [0] * batch, new
    total = [case["kv"] if i == 0 else _log_int(rng, min(16, case["kv"]), case["kv"]) for i in range(batch)]
    if case["mode"] == "decode":  # one token each, or a few drafted ones
        new = [min(case["new"], t) for t in total]
    else:  # one chunk among decoding requests
        new = [case["new"]] + [1] * (batch - 1)
    return [t - n for t, n in zip(total, new)], new


# ------------------------------------------------------------------------------------------------ inputs
def _pages(n: int, page: int) -> int:
    return -(-n // page)


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _filled_table(held: list[int], width: int, pool: torch.Tensor, page: int) -> tuple[torch.Tensor, int]:
    """A page table [batch, width] whose requests hold pages for ``held`` tokens, taken from the front of ``pool``; -1 elsewhere."""
    counts = [_pages(n, page) for n in held]
    table = torch.full((len(held), width), -1, dtype=torch.int32, device=DEV)
    rows = torch.repeat_interleave(torch.arange(len(held)), torch.tensor(counts))
    cols = torch.cat([torch.arange(c) for c in counts]) if counts else torch.empty(0, dtype=torch.long)
    table[rows.to(DEV), cols.to(DEV)] = pool[:sum(counts)]
    return table, sum(counts)


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16)

    if kind == "verify":
        rng = random.Random("drafts %s" % sorted((k, v) for k, v in case.items() if k != "name"))
        counts = [case["drafts"] if i == 0 else rng.randint(0, case["drafts"]) for i in range(case["batch"])]
        n, rows, vocab = sum(counts), sum(counts) + case["batch"], case["vocab"]
        cu = np.concatenate([[0], np.cumsum(counts)])
        target_rows = torch.tensor([cu[b] + b + i for b, c in enumerate(counts) for i in range(c)], dtype=torch.long, device=DEV)
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        logits = 2.5 * torch.randn(rows, vocab, generator=g, device=DEV)
        target = torch.softmax(logits, dim=-1).to(dtype)
        draft = torch.softmax(logits[target_rows] + 0.7 * torch.randn(n, vocab, generator=g, device=DEV), dim=-1).to(dtype)
        tokens = torch.multinomial(draft.float(), 1, generator=g).view(-1)
        return {"kind": kind, "target": target, "draft": draft if case["draft_probs"] else None, "tokens": tokens, "cu": _i32(cu.tolist()),
                "u": torch.rand(rows, generator=g, device=DEV), "most": case["drafts"]}

    page = case["page"]
    cached, new = _lengths(case)
    total = [c + n for c, n in zip(cached, new)]
    rows = sum(new) + case.get("pad", 0)
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    if kind in ("assign", "release"):
        width = _pages(max(total), page) + 3
        need = sum(_pages(t, page) for t in total)
        pool = torch.randperm(need + 29, generator=g, device=DEV).to(torch.int32)
        table, used = _filled_table(cached, width, pool, page)
        free = torch.full_like(pool, -1)
        free[:pool.numel() - used] = pool[used:]
        state = {"kind": kind, "page_table": table, "free_pages": free, "free_count": _i32([pool.numel() - used]), "cached": _i32(cached),
                 "page": page}
        if kind == "assign":
            return {**state, "new": _i32(new), "rows": rows}
        gone = torch.rand(len(cached), generator=g, device=DEV) < 0.5
        less = torch.randint(0, max(case["drop"], 1) + 1, (len(cached),), generator=g, device=DEV)
        keep = state["cached"] - less if case["drop"] else torch.where(gone, 0, state["cached"])
        return {**state, "keep": keep.clamp(min=0).to(torch.int32)}

    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    width = _pages(max(total), page)
    pool = torch.randperm(sum(_pages(t, page) for t in total) + 5, generator=g, device=DEV).to(torch.int32)
    table, _ = _filled_table(total, width, pool, page)
    k_cache, v_cache = randn(pool.numel(), page, hkv, d), randn(pool.numel(), page, hkv, d)
    state = {"kind": kind, "k_cache": k_cache, "v_cache": v_cache}
    if kind == "append":
        request = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(DEV)
        positions = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).to(DEV)
        slots = table[request, positions // page].long() * page + positions % page
        tail = rows - slots.numel()
        slots = torch.cat([slots, slots.new_full((tail,), -1)])
        positions = torch.cat([positions, positions.new_zeros(tail)]).to(torch.int32)
        angle = torch.outer(torch.arange(2048, device=DEV).double(), 10000.0 ** (-torch.arange(0, d, 2, device=DEV).double() / d))
        rope = torch.stack((angle.cos(), angle.sin()), dim=-1).to(torch.float32 if case["table"] == "fp32" else torch.bfloat16)
        return {**state, "qkv": randn(rows, (hq + 2 * hkv) * d), "rope": rope, "positions": positions, "slots": slots, "hq": hq,
                "q_out": torch.zeros(rows, hq, d, dtype=torch.bfloat16, device=DEV)}
    # scores of trained heads are peaked: a standard deviation of two in front of the softmax
    return {**state, "q": randn(rows, hq, d) * 2, "page_table": table, "kv_lens": _i32(total), "cu": _i32(cu),
            "out": torch.zeros(rows, hq, d, dtype=torch.bfloat16, device=DEV), "lens": (cached, new)}


# ------------------------------------------------------------------------------------------------ plain forms
def _assign_plain(s: dict):
    table, page, rows = s["page_table"], s["page"], s["rows"]
    cached, new = s["cached"].long().clamp(min=0), s["new"].long().clamp(min=0)
    have, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    ends = new.cumsum(0)
    fits = (ends <= rows) & (want <= table.size(1))
    need = torch.where(fits, want - have, 0)
    taken = need.cumsum(0)
    free = s["free_count"].long()
    granted = fits & ((need == 0) | (taken <= free))
    cols = torch.arange(table.size(1), device=DEV)
    fresh = granted[:, None] & (cols >= have[:, None]) & (cols < want[:, None])
    place = free - 1 - ((taken - need)[:, None] + cols - have[:, None])
    table.copy_(torch.where(fresh, s["free_pages"][place.clamp(0, s["free_pages"].numel() - 1)], table))
    row = torch.arange(rows, device=DEV)
    b = torch.searchsorted(ends, row, right=True)
    inside = b < new.numel()
    b = b.clamp(max=new.numel() - 1)
    held = inside & granted[b]
    pos = torch.where(held, cached[b] + row - (ends - new)[b], 0)
    entry = table[b, pos // page].long()
    slots = torch.where(held & (entry >= 0), entry * page + pos % page, -1)
    cu = torch.cat([ends.new_zeros(1), ends.clamp(max=rows)]).to(torch.int32)
    kv = torch.where(granted, cached + new, 0).to(torch.int32)
    lens = torch.where(granted, cached + new, cached).to(torch.int32)
    left = (free - torch.where(granted, need, 0).sum()).to(torch.int32)
    return table, cu, kv, lens, slots, pos.to(torch.int32), left


def _release_plain(s: dict):
    table, free_pages, page = s["page_table"], s["free_pages"], s["page"]
    lens = s["cached"].long().clamp(min=0)
    keep = torch.minimum(s["keep"].long().clamp(min=0), lens)
    have = ((lens + page - 1) // page).clamp(max=table.size(1))
    stay = ((keep + page - 1) // page).clamp(max=table.size(1))
    cols = torch.arange(table.size(1), device=DEV)
    back = table[(cols >= stay[:, None]) & (cols < have[:, None])]
    free = s["free_count"].long()
    free_pages[free + torch.arange(back.numel(), device=DEV)] = back
    return free_pages, (free + back.numel()).to(torch.int32)


def _rotate_plain(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    x = x.float().unflatten(-1, (-1, 2))
    c, s = cs[:, None, :, 0].float(), cs[:, None, :, 1].float()
    return torch.stack((x[..., 0] * c - x[..., 1] * s, x[..., 0] * s + x[..., 1] * c), dim=-1).flatten(-2).to(torch.bfloat16)


def _append_plain(s: dict):
    k_cache, v_cache, hq = s["k_cache"], s["v_cache"], s["hq"]
    hkv, d = k_cache.shape[2:]
    rows = (s["slots"] >= 0).nonzero().view(-1)
    q, k, v = s["qkv"][rows].view(rows.numel(), hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)
    cs, slots = s["rope"][s["positions"][rows].long()], s["slots"][rows]
    s["q_out"][rows] = _rotate_plain(q, cs)
    k_cache.view(-1, hkv, d)[slots] = _rotate_plain(k, cs)
    v_cache.view(-1, hkv, d)[slots] = v
    return s["q_out"], k_cache, v_cache


def _attend_plain(s: dict):
    out, page = s["out"], s["k_cache"].size(1)
    hkv, d = s["k_cache"].shape[2:]
    group = out.size(1) // hkv
    row = 0
    for b, (c, n) in enumerate(zip(*s["lens"])):
        if n == 0:
            continue
        ids = s["page_table"][b, :_pages(c + n, page)].long()
        k = s["k_cache"][ids].flatten(0, 1)[:c + n].transpose(0, 1).float()
        v = s["v_cache"][ids].flatten(0, 1)[:c + n].transpose(0, 1).float()
        step = max(1, (1 << 28) // (group * hkv * (c + n)))
        for t in range(0, n, step):
            m = min(step, n - t)
            q = s["q"][row + t:row + t + m].view(m, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, m * group, d).float()
            scores = (q @ k.transpose(1, 2)).view(hkv, m, group, c + n) * d ** -0.5
            seen = torch.arange(c + n, device=DEV) <= (c + t + torch.arange(m, device=DEV))[:, None]
            scores.masked_fill_(~seen[None, :, None, :], -math.inf)
            scores -= scores.amax(dim=-1, keepdim=True)
            scores.exp_()
            o = (scores.view(hkv, m * group, c + n) @ v).view(hkv, m, group, d) / scores.sum(dim=-1, keepdim=True)
            out[row + t:row + t + m] = o.permute(1, 0, 2, 3).reshape(m, hkv * group, d).to(out.dtype)
        row += n
    return out


def _verify_plain(s: dict):
    target, draft, tokens, cu, u, most = s["target"], s["draft"], s["tokens"], s["cu"].long(), s["u"].double(), s["most"]
    batch = cu.numel() - 1
    b, i = torch.arange(batch, device=DEV), torch.arange(most, device=DEV)
    count = cu[1:] - cu[:-1]
    there = i < count[:, None]
    at = (cu[:-1, None] + i).clamp(max=max(tokens.numel() - 1, 0))
    x = tokens[at]
    row = (cu[:-1] + b)[:, None] + i
    row = torch.where(there, row, 0)
    p = target[row, x].double()
    q = draft[at, x].double() if draft is not None else torch.ones_like(p)
    good = there & (u[row] * q < p)
    accepted = good.long().cumprod(dim=1).sum(dim=1)
    refused = accepted < count
    last = target[cu[:-1] + b + accepted].double()
    at = (cu[:-1] + accepted).clamp(max=max(tokens.numel() - 1, 0))
    if draft is not None:
        rest = (last - draft[at].double()).clamp(min=0)
    else:
        rest = last.scatter(1, tokens[at][:, None], 0.0)
    weights = torch.where(refused[:, None], rest, last)
    weights = torch.where(weights.sum(dim=1, keepdim=True) > 0, weights, last)
    sums = weights.cumsum(dim=1)
    aim = u[cu[1:] + b] * sums[:, -1]
    token = (sums <= aim[:, None]).sum(dim=1)
    vocab = torch.arange(target.size(1), device=DEV)
    token = torch.minimum(token, torch.where(weights > 0, vocab, 0).amax(dim=1))
    j = torch.arange(most + 1, device=DEV)
    drafted = torch.cat([x, x.new_zeros(batch, 1)], dim=1)
    result = torch.where(j < accepted[:, None], drafted, torch.where(j == accepted[:, None], token[:, None], -1))
    return result, accepted.to(torch.int32)


# ------------------------------------------------------------------------------------------------ the call
@torch.inference_mode()
def run(s: dict):
    kind = s["kind"]
    if not own:
        return {"assign": _assign_plain, "release": _release_plain, "append": _append_plain, "attend": _attend_plain, "verify": _verify_plain}[kind](s)
    import quest_b200 as quest
    if kind == "assign":
        step = quest.page_assign(s["page_table"], s["free_pages"], s["free_count"], s["cached"], s["new"], s["rows"], s["page"])
        return s["page_table"], step.cu_new, step.kv_lens, step.lens, step.slots, step.positions, step.free_count
    if kind == "release":
        left = quest.page_release(s["page_table"], s["free_pages"], s["free_count"], s["cached"], s["keep"], s["page"])
        return s["free_pages"], left
    if kind == "append":
        quest.rope_paged_append(s["qkv"], s["rope"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["hq"], q_out=s["q_out"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    if kind == "attend":
        return quest.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"], s["cu"], out=s["out"])
    return quest.verify_drafts(s["target"], s["tokens"], s["cu"], s["u"], s["most"], draft_probs=s["draft"])


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "verify":  # one or two rows of probabilities for each sampled token; one value of either for each draft
        size = 4 if case["dtype"] == "fp32" else 2
        b, v, n = case["batch"], case["vocab"], case["batch"] * case["drafts"] / 2
        return {"bytes": b * v * size * (1.5 if case["draft_probs"] else 1) + n * (8 + 4 + 2 * size) + b * (8 * (case["drafts"] + 1) + 8), "flops": 2 * b * v}
    cached, new = _lengths(case)
    page, b, t = case["page"], case["batch"], sum(new) + case.get("pad", 0)
    if kind == "assign":
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        return {"bytes": 4 * 5 * b + 8 * fresh + 12 * t, "flops": 4 * b + 4 * t}
    if kind == "release":  # every second request as a whole, or the few pages behind refused drafts
        back = sum(_pages(c, page) for c in cached) / 2 if case["drop"] == 0 else b * case["drop"] / 2 / page
        return {"bytes": 8 * b + 8 * back, "flops": 4 * b}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if kind == "append":
        positions = len({p for c, n in zip(cached, new) for p in range(c, c + n)})
        return {"bytes": 4 * sum(new) * (hq + 2 * hkv) * d + 12 * t + positions * d * (4 if case["table"] == "fp32" else 2), "flops": 3 * sum(new) * (hq + hkv) * d}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    keys = sum(c + n for c, n in zip(cached, new) if n)
    return {"bytes": 4 * keys * hkv * d + 4 * sum(new) * hq * d + 8 * b + 4 * keys / page, "flops": 4 * seen * hq * d}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def _exact_pages(case: dict, s: dict):
    """Request by request, page by page, on the host."""
    table, free_pages = s["page_table"].cpu().numpy().copy(), s["free_pages"].cpu().numpy().copy()
    free, page, cached = int(s["free_count"]), s["page"], s["cached"].tolist()
    if case["kind"] == "release":
        for b, (n, keep) in enumerate(zip(cached, s["keep"].tolist())):
            for j in range(_pages(keep, page), _pages(n, page)):
                free_pages[free] = table[b, j]
                free += 1
        return torch.from_numpy(free_pages), torch.tensor([free], dtype=torch.int32)
    cu, kv, lens, slots, positions = [0], [], [], [-1] * s["rows"], [0] * s["rows"]
    start = 0
    for b, (c, n) in enumerate(zip(cached, s["new"].tolist())):
        for j in range(_pages(c, page), _pages(c + n, page)):  # rows, pages and width suffice in these cases
            free -= 1
            table[b, j] = free_pages[free]
        for i in range(n):
            positions[start + i] = c + i
            slots[start + i] = int(table[b, (c + i) // page]) * page + (c + i) % page
        start += n
        cu.append(start), kv.append(c + n), lens.append(c + n)
    as_i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return torch.from_numpy(table), as_i32(cu), as_i32(kv), as_i32(lens), torch.tensor(slots), as_i32(positions), as_i32([free])


def _exact_verify(s: dict):
    target, draft, u, cu, most = s["target"], s["draft"], s["u"].double().cpu().numpy(), s["cu"].tolist(), s["most"]
    tokens = s["tokens"].tolist()
    result, accepted = [], []
    for b in range(len(cu) - 1):
        first, n = cu[b] + b, cu[b + 1] - cu[b]
        i = 0
        while i < n:
            x = tokens[cu[b] + i]
            q = 1.0 if draft is None else float(draft[cu[b] + i, x])
            if not u[first + i] * q < float(target[first + i, x]):
                break
            i += 1
        w = target[first + i].double().cpu().numpy()
        if i < n:
            rest = w.copy()
            if draft is None:
                rest[tokens[cu[b] + i]] = 0
            else:
                rest = np.maximum(w - draft[cu[b] + i].double().cpu().numpy(), 0)
            w = rest if rest.sum() > 0 else w
        sums = np.cumsum(w)
        t = min(int(np.searchsorted(sums, u[first + n] * sums[-1], side="right")), int(np.flatnonzero(w)[-1]))
        accepted.append(i)
        result.append(tokens[cu[b]:cu[b] + i] + [t] + [-1] * (most - i))
    return torch.tensor(result), torch.tensor(accepted, dtype=torch.int32)


@torch.inference_mode()
def exact(case: dict, seed: int):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind in ("assign", "release"):
        return _exact_pages(case, s)
    if kind == "verify":
        return _exact_verify(s)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    group = case["hq"] // hkv
    if kind == "append":
        q_out, k_cache, v_cache = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
        turn = torch.view_as_complex(s["rope"].double().contiguous())
        x = s["qkv"].double().view(-1, case["hq"] + 2 * hkv, d)
        for i in range(0, x.size(0), 4096):
            slots = s["slots"][i:i + 4096]
            live = slots >= 0
            heads = x[i:i + 4096][live]
            z = torch.view_as_complex(heads[:, :-hkv].reshape(heads.size(0), -1, d // 2, 2)) * turn[s["positions"][i:i + 4096][live].long()][:, None]
            z = torch.view_as_real(z).flatten(-2)
            q_out[i:i + 4096][live] = z[:, :case["hq"]]
            k_cache[slots[live] // page, slots[live] % page] = z[:, case["hq"]:]
            v_cache[slots[live] // page, slots[live] % page] = heads[:, -hkv:]
        return q_out, k_cache, v_cache
    if work(case)["flops"] > 3e13:
        return None
    out = s["out"].double()
    row = 0
    for b, (c, n) in enumerate(zip(*s["lens"])):
        key = torch.arange(c + n, device=DEV)
        place = s["page_table"][b].long()[key // page]
        for h in range(hkv):
            k, v = s["k_cache"][place, key % page, h].double(), s["v_cache"][place, key % page, h].double()
            step = max(1, (1 << 27) // (group * (c + n)))
            for t in range(0, n, step):
                m = min(step, n - t)
                q = s["q"][row + t:row + t + m, h * group:(h + 1) * group].double()
                a = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
                a = a.masked_fill((key > c + t + torch.arange(m, device=DEV)[:, None])[:, None], -math.inf)
                out[row + t:row + t + m, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", torch.softmax(a, dim=-1), v)
        row += n
    return out
