"""The 64-bit host implementations that the serving operators are compared with, against other ways to the same answers."""
from __future__ import annotations

import itertools
import random

import numpy as np
import pytest
import torch

import paged_reference as ref


@pytest.mark.parametrize("seed", range(6))
def test_assign_and_release_move_pages_between_the_stack_and_the_requests(seed):
    """Steps of random lengths: no page is held twice or lost, a token's slot stays where it was, what was refused holds what it held."""
    rng = random.Random(seed)
    batch, page, width, pages = rng.randint(1, 9), rng.choice([1, 3, 16]), 6, rng.randint(4, 30)
    table, stack, free = np.full((batch, width), -1), list(range(pages)), pages
    lens, where = [0] * batch, {}
    for _ in range(12):
        new = [rng.choice([0, 1, rng.randint(0, 2 * page)]) for _ in range(batch)]
        rows = max(0, sum(new) + rng.choice([0, 2, -3]))
        table, cu, kv, after, slots, positions, left = ref.assign(table, stack, free, lens, new, rows, page)
        assert cu[0] == 0 and len(slots) == len(positions) == rows
        for b in range(batch):
            granted = after[b] == lens[b] + new[b] and kv[b] == after[b]
            assert granted or (after[b] == lens[b] and kv[b] == 0)
            mine = slots[cu[b]:cu[b + 1]]
            if granted:
                assert positions[cu[b]:cu[b + 1]] == list(range(lens[b], after[b])) and cu[b + 1] - cu[b] == new[b]
                where.update({(b, lens[b] + i): s for i, s in enumerate(mine)})
            else:
                assert all(s == -1 for s in mine)
        assert all(s == -1 for s in slots[cu[-1]:])
        lens, free = after, left
        held = [int(table[b, j]) for b in range(batch) for j in range(ref.ceil_div(lens[b], page))]
        assert sorted(held + list(stack[:free])) == list(range(pages))
        for (b, position), slot in where.items():
            assert slot == table[b, position // page] * page + position % page
        keep = [rng.choice([n, n, max(n - 2, 0), 0]) for n in lens]
        stack, free = ref.release(table, stack, free, lens, keep, page)
        stack = list(stack)
        lens = keep
        where = {(b, i): s for (b, i), s in where.items() if i < lens[b]}
        held = [int(table[b, j]) for b in range(batch) for j in range(ref.ceil_div(lens[b], page))]
        assert sorted(held + stack[:free]) == list(range(pages))


def test_assign_refuses_in_order():
    table = np.full((4, 2), -1)
    # the second needs three entries of two, the third the last page, so that the fourth, whose page has room, is served all the same
    table[3, 0] = 9
    got = ref.assign(table, [4, 5], 2, [0, 0, 0, 3], [4, 12, 5, 1], 40, 4)
    assert got[2] == [4, 0, 0, 4] and got[3] == [4, 0, 0, 4] and got[6] == 1 and got[1] == [0, 4, 16, 21, 22]
    assert got[4][:4] == [20, 21, 22, 23] and got[4][4:21] == [-1] * 17 and got[4][21] == 39


@pytest.mark.parametrize("hq, hkv, d, page", [(4, 2, 64, 16), (3, 1, 8, 5), (2, 2, 16, 1)])
def test_attention_is_the_masked_dense_one(hq, hkv, d, page):
    """All rows of a request at once over dense keys and values, scores behind a row's own token at minus infinity."""
    kv, new = [7, 0, 40, 23, 2], [3, 2, 1, 23, 5]
    s = ref.paged_state(hq + d, kv, new, hq, hkv, d, page, pad=2, device="cpu")
    before = torch.full(s["q"].shape, 5.0)
    got, size = ref.attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], kv, s["cu_new"].tolist(), 0.3, before)
    assert (got[sum(new):] == 5).all()
    for b, (n, k) in enumerate(zip(new, kv)):
        rows = slice(sum(new[:b]), sum(new[:b + 1]))
        if k == 0:
            assert (got[rows] == 0).all()
            continue
        slots = (s["page_table"][b, :ref.ceil_div(k, page)].long()[:, None] * page + torch.arange(page)).view(-1)[:k]
        keys, values = (x.double().flatten(0, 1)[slots].repeat_interleave(hq // hkv, dim=1) for x in (s["k_cache"], s["v_cache"]))
        scores = torch.einsum("thd,jhd->thj", s["q"][rows].double(), keys) * 0.3
        hidden = torch.arange(k)[None] > torch.arange(k - n, k)[:, None]
        p = torch.softmax(scores.masked_fill(hidden[:, None], float("-inf")), dim=-1).nan_to_num(0)  # rows in front of the first key
        assert (got[rows] - torch.einsum("thj,jhd->thd", p, values)).abs().max() < 1e-13
        assert (size[rows] - torch.einsum("thj,jhd->thd", p, values.abs())).abs().max() < 1e-13


@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_gives_the_first_token_the_distribution_of_the_target(with_draft):
    """Every draft token weighted with its probability and both uniforms on a grid: what comes out first has the target's
    probabilities, up to the grid's step at each border."""
    p, q = torch.tensor([0.5, 0.25, 0.125, 0.125, 0.0]), torch.tensor([0.125, 0.5, 0.25, 0.0, 0.125])
    n = 64
    grid = [(i + 0.5) / n for i in range(n)]
    share = torch.zeros(5, dtype=torch.float64)
    for x in range(5):
        weight = q[x].item() if with_draft else float(x == 1)  # without probabilities: a draft that always is the same token
        if weight == 0:
            continue
        pairs = list(itertools.product(grid, grid))
        u = torch.tensor(pairs).view(-1)
        trials = len(pairs)
        target, draft = p.expand(2 * trials, 5), q.expand(trials, 5) if with_draft else None
        tokens, accepted = ref.verify(target, draft, [x] * trials, list(range(trials + 1)), u, 1)
        for t, k in zip(tokens, accepted):
            assert (t[0] == x) if k else (t[1] == -1)
            share[t[0]] += weight / trials
    assert (share - p).abs().max() <= 5 / n


def test_verify_stops_at_the_first_refusal_and_draws_behind_the_last_draft():
    rows = torch.tensor([[0.5, 0.5, 0.0], [0.0, 0.5, 0.5], [0.25, 0.25, 0.5], [1.0, 0.0, 0.0]])
    draft = torch.tensor([[1.0, 0.0, 0.0], [0.0, 0.0, 1.0], [0.0, 0.0, 1.0]])
    u = torch.tensor([0.25, 0.25, 0.25, 0.25])
    assert ref.verify(rows, draft, [0, 2, 2], [0, 3], u, 3) == ([[0, 2, 2, 0]], [3])
    assert ref.verify(rows, draft, [0, 2, 2], [0, 3], u, 2) == ([[0, 2, 1]], [2])          # the third draft is not looked at: drawn from its row
    assert ref.verify(rows, draft, [0, 2, 2], [0, 3], torch.tensor([0.25, 0.75, 0.0, 0.9]), 3) == ([[0, 1, -1, -1]], [1])  # what is left of the second row
    assert ref.verify(rows, draft, [0, 7, 2], [0, 3], u, 3)[1] == [1]
    assert ref.verify(rows[:1], None, [], [0, 0], torch.tensor([0.5]), 1) == ([[1, -1]], [0])
