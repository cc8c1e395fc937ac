"""Plain 64-bit host implementations of the serving operators, and random states for them."""
from __future__ import annotations

import numpy as np
import torch


def ceil_div(a: int, b: int) -> int:
    return -(-a // b)


def assign(table, free_pages, free, cached, new, rows, page):
    """Request by request.  Returns (page table, cu, kv_lens, lens, slots, positions, free count) as lists / arrays."""
    table = np.array(table, copy=True)
    width = table.shape[1]
    cu, kv, lens, slots, positions = [0], [], [], [-1] * rows, [0] * rows
    end = spent = 0
    exhausted = False  # once a request has found too few pages, later ones that need any are refused, too
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        start, end = end, end + n
        have, want = ceil_div(c, page), ceil_div(c + n, page)
        granted = end <= rows and want <= width
        need = want - have if granted else 0
        if granted and need > 0:
            if exhausted or spent + need > free:
                exhausted, granted = True, False
            else:
                for i in range(need):
                    table[b, have + i] = free_pages[free - 1 - spent - i]
                spent += need
        if granted:
            for i in range(n):
                entry = int(table[b, (c + i) // page])
                positions[start + i] = c + i
                slots[start + i] = entry * page + (c + i) % page if entry >= 0 else -1
        cu.append(min(end, rows)), kv.append(c + n if granted else 0), lens.append(c + n if granted else c)
    return table, cu, kv, lens, slots, positions, free - spent


def release(table, free_pages, free, lens, keep, page):
    free_pages = np.array(free_pages, copy=True)
    for b, (n, k) in enumerate(zip(lens, keep)):
        n = max(n, 0)
        k = min(max(k, 0), n)
        for j in range(min(ceil_div(k, page), table.shape[1]), min(ceil_div(n, page), table.shape[1])):
            if free < len(free_pages):
                free_pages[free] = table[b, j]
                free += 1
    return free_pages, free


def attention(q, k_cache, v_cache, table, kv_lens, cu, scale, out):
    """(out, weight of the values' magnitudes sum_j p_j |v_j|) in float64; rows outside every request keep ``out``."""
    q, k_cache, v_cache, out = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu(), out.double().cpu().clone()
    size = torch.zeros_like(out)
    page, hkv = k_cache.shape[1:3]
    group = q.shape[1] // hkv
    for b, kv in enumerate(kv_lens):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            continue
        out[cu[b]:cu[b + 1]] = 0
        if kv == 0:
            continue
        j = torch.arange(kv)
        at = torch.as_tensor(table[b]).long()[j // page]
        k, v = k_cache[at, j % page], v_cache[at, j % page]
        for t in range(n):
            seen = kv - n + t + 1
            if seen <= 0:
                continue
            s = torch.einsum("hgd,jhd->hgj", q[cu[b] + t].view(hkv, group, -1), k[:seen]) * scale
            p = torch.softmax(s, dim=-1)
            out[cu[b] + t] = torch.einsum("hgj,jhd->hgd", p, v[:seen]).reshape(hkv * group, -1)
            size[cu[b] + t] = torch.einsum("hgj,jhd->hgd", p, v[:seen].abs()).reshape(hkv * group, -1)
    return out, size


def verify(target, draft, tokens, cu, u, most):
    target = target.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    u = u.double().cpu().numpy()
    vocab = target.shape[1]
    result, accepted = [], []
    for b in range(len(cu) - 1):
        first, drafts = cu[b] + b, cu[b + 1] - cu[b]
        kept, stop = 0, min(drafts, most)
        while kept < stop:
            x = tokens[cu[b] + kept]
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else draft[cu[b] + kept, x]
            if not u[first + kept] * q < target[first + kept, x]:
                break
            kept += 1
        p = target[first + kept]
        w = np.where(p > 0, p, 0)
        if kept < stop:
            if draft is not None:
                r = p - draft[cu[b] + kept]
                r = np.where(r > 0, r, 0)
            else:
                r = w.copy()
                if 0 <= tokens[cu[b] + kept] < vocab:
                    r[tokens[cu[b] + kept]] = 0
            w = r if r.sum() > 0 else w
        total = np.cumsum(w)
        positive = np.flatnonzero(w)
        t = int(np.searchsorted(total, u[first + drafts] * total[-1], side="right"))
        t = min(t, int(positive[-1]) if positive.size else 0)
        accepted.append(kept)
        result.append(list(tokens[cu[b]:cu[b] + kept]) + [t] + [-1] * (most - kept))
    return result, accepted


def paged_state(seed, kv_lens, new_lens, hq, hkv, d, page, pad=0, spread=1.0, device="cuda"):
    """Requests of those lengths over a shuffled pool.  Pages and places that hold no token are NaN, table entries behind a
    request's pages point nowhere."""
    g = torch.Generator().manual_seed(seed)
    counts = [ceil_div(n, page) for n in kv_lens]
    pool = torch.randperm(sum(counts) + 3, generator=g)
    width = max(counts + [1]) + 1
    table = torch.full((len(kv_lens), width), -7, dtype=torch.int32)
    k = torch.full((pool.numel(), page, hkv, d), float("nan"), dtype=torch.bfloat16)
    v = k.clone()
    used = 0
    for b, n in enumerate(kv_lens):
        ids = pool[used:used + counts[b]]
        table[b, :counts[b]] = ids.int()
        used += counts[b]
        for i, page_id in enumerate(ids.tolist()):
            live = min(page, n - i * page)
            k[page_id, :live] = torch.randn(live, hkv, d, generator=g).to(torch.bfloat16)
            v[page_id, :live] = torch.randn(live, hkv, d, generator=g).to(torch.bfloat16)
    cu = np.concatenate([[0], np.cumsum(new_lens)]).astype(int).tolist()
    q = (torch.randn(cu[-1] + pad, hq, d, generator=g) * spread).to(torch.bfloat16)
    as_i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=q.to(device), k_cache=k.to(device), v_cache=v.to(device), page_table=table.to(device), kv_lens=as_i32(kv_lens), cu_new=as_i32(cu))
