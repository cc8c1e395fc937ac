"""The serving operators on the GPU against plain 64-bit implementations."""
from __future__ import annotations

import os
import random
import subprocess
import sys
import threading

import pytest
import torch

import paged_reference as ref
import quest_b200 as quest
from quest_b200.prefill import rope_table

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ page tables
def assign_case(seed, batch, page, width, most_cached, most_new, free, rows_less=0):
    rng = random.Random(seed)
    cached = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, most_cached)]) for _ in range(batch)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(batch)]
    cached = [min(c, width * page) for c in cached]
    pool = list(range(batch * width + free))
    rng.shuffle(pool)
    table = torch.full((batch, width), -1, dtype=torch.int32)
    for b, c in enumerate(cached):
        for j in range(ref.ceil_div(c, page)):
            table[b, j] = pool.pop()
    free_pages = pool[:free] + [-1] * 5
    rows = max(0, sum(new) + rng.choice([0, 3]) - rows_less)
    return table, free_pages, free, cached, new, rows


@pytest.mark.parametrize("batch, page, width, most_cached, most_new, free, rows_less", [
    (1, 16, 4, 20, 30, 9, 0),
    (1, 16, 4, 0, 0, 0, 0),
    (7, 1, 9, 4, 4, 60, 0),
    (33, 16, 20, 200, 90, 400, 0),
    (33, 16, 20, 200, 90, 37, 0),      # the pages run out
    (33, 48, 3, 140, 90, 400, 0),      # table rows run out
    (40, 16, 20, 100, 90, 900, 500),   # rows run out
    (512, 32, 5, 100, 40, 2000, 0),
    (513, 64, 5, 100, 40, 900, 3),
    (1500, 16, 6, 60, 30, 5000, 0),
    (8192, 16, 2, 20, 3, 9000, 0),
])
def test_page_assign(batch, page, width, most_cached, most_new, free, rows_less):
    table, free_pages, free, cached, new, rows = assign_case(batch + page, batch, page, width, most_cached, most_new, free, rows_less)
    t, cu, kv, lens, slots, positions, left = ref.assign(table.numpy(), free_pages, free, cached, new, rows, page)
    dev = table.cuda()
    step = quest.page_assign(dev, i32(free_pages), i32([free]), i32(cached), i32(new), rows, page)
    assert step.cu_new.tolist() == cu and step.kv_lens.tolist() == kv and step.lens.tolist() == lens
    assert step.slots.tolist() == slots and step.positions.tolist() == positions and step.free_count.tolist() == [left]
    assert torch.equal(dev.cpu(), torch.from_numpy(t))
    live = [s for s in slots if s >= 0]
    assert len(set(live)) == len(live)


def test_page_assign_takes_negative_and_large_lengths():
    table = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    step = quest.page_assign(table, i32([5, 6, 7]), i32([3]), i32([-4, 2**31 - 1, 16, 0]), i32([1, 2**31 - 1, -3, 16]), 40, 16)
    assert step.kv_lens.tolist() == [1, 0, 0, 0] and step.cu_new.tolist() == [0, 1, 40, 40, 40]  # the rows end with the second
    assert step.lens.tolist() == [1, 2**31 - 1, 16, 0] and step.free_count.tolist() == [2]


def test_page_assign_without_requests_or_rows():
    step = quest.page_assign(i32([]).view(0, 3), i32([1, 2]), i32([2]), i32([]), i32([]), 5, 16)
    assert step.cu_new.tolist() == [0] and step.slots.tolist() == [-1] * 5 and step.positions.tolist() == [0] * 5 and step.free_count.tolist() == [2]
    step = quest.page_assign(i32([[1]]), i32([1, 2]), i32([2]), i32([3]), i32([0]), 0, 16)
    assert step.cu_new.tolist() == [0, 0] and step.kv_lens.tolist() == [3] and step.slots.numel() == 0


@pytest.mark.parametrize("batch, page, width, capacity", [(1, 16, 4, 50), (9, 1, 30, 300), (100, 16, 40, 5000), (700, 64, 9, 7000), (100, 16, 40, 60), (8192, 16, 2, 20000)])
def test_page_release(batch, page, width, capacity):
    rng = random.Random(batch)
    lens = [rng.randint(-1, width * page) for _ in range(batch)]
    keep = [rng.choice([0, n, n - 1, n // 2, n + 5]) for n in lens]
    table = torch.arange(batch * width, dtype=torch.int32).view(batch, width)
    free_pages, free = [-9] * capacity, min(13, capacity)
    want, left = ref.release(table.numpy(), free_pages, free, lens, keep, page)
    pages = i32(free_pages)
    count = quest.page_release(table.cuda(), pages, i32([free]), i32(lens), i32(keep), page)
    assert count.tolist() == [left] and pages.tolist() == want.tolist()


# ------------------------------------------------------------------------------------------------ rotary embedding into the pages
@pytest.mark.parametrize("rows, hq, hkv, d, page, table_dtype", [
    (1, 1, 1, 64, 16, torch.float32), (5, 16, 16, 128, 64, torch.bfloat16), (33, 28, 4, 64, 16, torch.bfloat16), (130, 8, 1, 128, 128, torch.float32),
    (7, 3, 3, 8, 5, torch.float32), (19, 4, 2, 80, 32, torch.float32)])
@pytest.mark.parametrize("layout", ["tokens", "heads", "pair"])
def test_rope_paged_append(rows, hq, hkv, d, page, table_dtype, layout):
    g = torch.Generator().manual_seed(rows)
    pages = ref.ceil_div(rows, page) + 3
    wide = torch.randn(rows, (hq + 2 * hkv) * d + 16, generator=g).to(torch.bfloat16)
    qkv = wide.cuda()[:, 8:-8]  # a view into a wider buffer
    table = rope_table(d, 300).to(table_dtype)
    positions = torch.randint(0, 300, (rows,), generator=g).int()
    slots = torch.randperm(pages * page, generator=g)[:rows]
    if layout == "tokens":
        k_cache, v_cache = (torch.full((pages, page, hkv, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    elif layout == "heads":
        k_cache, v_cache = (torch.full((pages, hkv, page, d), 7.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        k_cache, v_cache = torch.full((pages, 2, page, hkv, d), 7.0, dtype=torch.bfloat16, device="cuda").unbind(1)
    if rows > 4:  # rows that are not to be stored
        slots[1], slots[2], positions[3], positions[4] = -1, pages * page, 300, -1
    skipped = [1, 2, 3, 4] if rows > 4 else []
    q_out = torch.full((rows, hq, d), 3.0, dtype=torch.bfloat16, device="cuda")
    got = quest.rope_paged_append(qkv, table.cuda(), positions.cuda(), slots.cuda(), k_cache, v_cache, hq, q_out=q_out)
    assert got is q_out

    q, k, v = wide[:, 8:-8].reshape(rows, hq + 2 * hkv, d).split((hq, hkv, hkv), dim=1)
    cs = table[positions.long().clamp(0, 299)]
    rot = lambda x: _rotate(x, cs)  # noqa: E731
    want_q, want_k, want_v = torch.full((rows, hq, d), 3.0, dtype=torch.bfloat16), torch.full((pages, page, hkv, d), 7.0, dtype=torch.bfloat16), torch.full((pages, page, hkv, d), 7.0, dtype=torch.bfloat16)
    for r in range(rows):
        if r in skipped:
            continue
        s = int(slots[r])
        want_q[r], want_k[s // page, s % page], want_v[s // page, s % page] = rot(q)[r], rot(k)[r], v[r]
    assert torch.equal(q_out.cpu(), want_q) and torch.equal(k_cache.cpu(), want_k) and torch.equal(v_cache.cpu(), want_v)


def _rotate(x, cs):
    xf = x.float().unflatten(-1, (-1, 2))
    c, s = cs[:, None, :, 0].float(), cs[:, None, :, 1].float()
    return torch.stack((xf[..., 0] * c - xf[..., 1] * s, xf[..., 0] * s + xf[..., 1] * c), dim=-1).flatten(-2).to(x.dtype)


# ------------------------------------------------------------------------------------------------ attention
def check_attention(s, scale=None, out=None):
    """Tolerance: the scores' sums in fp32 over products that are exact move a probability by less than 2^-10 of itself at these
    sizes (128 products of magnitude up to about 50, scaled by 0.09, at 2^-23 each: below 2^-12), its rounding to bf16 for the
    second product by 2^-8, so the output by (2^-8 + 2^-10) sum p|v|; its own rounding to bf16 adds 2^-8 of it."""
    q = s["q"]
    if out is None:
        out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
    want, size = ref.attention(q, s["k_cache"], s["v_cache"], s["page_table"].cpu(), s["kv_lens"].tolist(), s["cu_new"].tolist(),
                               q.size(2) ** -0.5 if scale is None else scale, out)
    got = quest.paged_attention(**s, scale=scale, out=out)
    assert got is out
    got = got.double().cpu()
    error = (got - want).abs()
    allowed = (2 ** -8 + 2 ** -10) * size + 2 ** -8 * want.abs() + 1e-30
    worst = (error / allowed).max().item() if error.numel() else 0
    assert torch.isfinite(got).all() and worst <= 1, (worst, (error > allowed).nonzero()[:4].tolist())


HEADS = [(1, 1), (16, 16), (64, 8), (28, 4), (5, 5), (12, 2), (8, 1)]


@pytest.mark.parametrize("hq, hkv", HEADS)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_single_tokens(hq, hkv, d):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 300]
    check_attention(ref.paged_state(hq * d, lens, [1] * len(lens), hq, hkv, d, 16, spread=2.0))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_pages(page, d):
    lens = [1, page - 1, page, page + 1, 2 * page + 3, 400]
    check_attention(ref.paged_state(page + d, lens, [1, 3, page, 2, 70, 150], 4, 2, d, page, pad=2))


@pytest.mark.parametrize("hq, hkv", [(2, 2), (8, 1), (7, 1), (12, 2), (40, 2)])
@pytest.mark.parametrize("new", [1, 2, 5, 31, 127, 128, 129, 300])
def test_attention_chunks(hq, hkv, new):
    lens = [new, new + 1, new + 100, new + 200]
    check_attention(ref.paged_state(new + hq, lens, [new] * 4, hq, hkv, 128 if new % 2 else 64, 16))


def test_attention_mixed_batch_with_empty_and_refused_requests():
    kv, new = [200, 0, 0, 77, 513, 5, 300, 1], [1, 0, 9, 77, 130, 0, 3, 1]
    s = ref.paged_state(3, kv, new, 8, 2, 128, 32, pad=11)
    check_attention(s)


def test_attention_rows_before_the_first_key():
    """More new rows than tokens held (a caller whose kv_lens are behind): the rows that see no key give zeros."""
    s = ref.paged_state(4, [3, 40, 130], [8, 300, 131], 4, 4, 64, 16)
    check_attention(s)


def test_attention_long_context_is_split_and_joined():
    s = ref.paged_state(5, [5000, 1, 3001], [1, 1, 2], 8, 2, 128, 64)
    check_attention(s)
    s = ref.paged_state(6, [9000], [130], 2, 1, 64, 128)
    check_attention(s)


def test_attention_strides_and_scale():
    s = ref.paged_state(7, [100, 200], [20, 1], 6, 3, 128, 16)
    pages = s["k_cache"].size(0)
    both = torch.zeros(pages, 2, 3, 16, 128, dtype=torch.bfloat16, device="cuda").transpose(2, 3)  # heads before tokens, k and v in one pool
    both[:, 0].copy_(s["k_cache"]), both[:, 1].copy_(s["v_cache"])
    s["k_cache"], s["v_cache"] = both[:, 0], both[:, 1]
    wide = torch.zeros(21, 9, 136, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:8, 8:].copy_(s["q"])
    s["q"] = wide[:, 2:8, 8:]
    out = torch.full((21, 10, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    check_attention(s, scale=0.2, out=out[:, 1:7])
    assert (out[:, 0] == 5).all() and (out[:, 7:] == 5).all()


def test_attention_of_extreme_scores():
    """Scores of several hundreds, a first tile that is far below a later one, and equal keys."""
    s = ref.paged_state(8, [600, 300], [3, 2], 2, 1, 128, 16)
    s["q"].mul_(8)
    page = s["page_table"][0, 20].long()
    s["k_cache"][page] *= 4
    s["k_cache"][s["page_table"][1, :18].long()] = 0.5
    want, size = ref.attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"].cpu(), s["kv_lens"].tolist(), s["cu_new"].tolist(), 128 ** -0.5, s["q"])
    got = quest.paged_attention(**s).double().cpu()
    # scores up to 400: sums of magnitude up to 5000 before the scale move by 128 * 2^-23 * 5000 * 0.09 = 2^-7 at the very most
    assert ((got - want).abs() <= (2 ** -8 + 2 ** -7) * size + 2 ** -8 * want.abs()).all()


def scores_case(profile, d, hq=4, hkv=2, new=3):
    """A request whose score at key j is near profile[j] for every row (natural units): queries along one direction."""
    kv, page = len(profile), 64
    g = torch.Generator().manual_seed(kv + d)
    u = torch.randn(d, generator=g)
    u /= u.norm()
    pages = ref.ceil_div(kv, page)
    q = (d ** 0.5 * u + 0.02 * torch.randn(new, hq, d, generator=g)).bfloat16().cuda()  # scale q.k is then u.k
    k = torch.tensor(profile)[:, None, None] * u + 0.02 * torch.randn(kv, hkv, d, generator=g)
    cache = torch.zeros(2, pages * page, hkv, d)
    cache[0, :kv], cache[1, :kv] = k, torch.randn(kv, hkv, d, generator=g)
    k_cache, v_cache = cache.bfloat16().cuda().view(2, pages, page, hkv, d).unbind(0)
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, page_table=torch.arange(pages, dtype=torch.int32, device="cuda")[None], kv_lens=i32([kv]),
                cu_new=i32([0, new]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [3, 200])
@pytest.mark.parametrize("name", ["rise", "fall", "leap", "slope", "spikes", "plateau", "waves"])
def test_attention_follows_the_maximum_from_step_to_step(name, new, d):
    """Scores that grow or fall between steps, by a little, by what fp32 can no longer hold, and at single keys of any place in a
    step.  With scores up to 250 their sums in fp32 (128 products of at most about 40, of both signs) are off by less than 2^-14, as
    check_attention allows for; bf16 queries and keys make the scores themselves uneven, which the oracle sees, too."""
    kv = 128 * 9 + 40
    profile = {
        "rise": [j // 128 * 3.0 for j in range(kv)],  # 2^4.3 a step: the sum passes its limit every few steps
        "fall": [30.0 - j // 128 * 9.0 for j in range(kv)],
        "leap": [-120.0 if j < 500 else 120.0 for j in range(kv)],  # 2^346 at once
        "slope": [-200.0 + 400.0 * j / kv for j in range(kv)],
        "spikes": [25.0 + j / 100 if j % 131 == 14 else 0.0 for j in range(kv)],
        "plateau": [0.0 if j < 128 else 4.9 for j in range(kv)],  # 128 weights of 2^7
        "waves": [60.0 if j // 128 % 2 else -60.0 for j in range(kv)],
    }[name]
    check_attention(scores_case(profile, d, new=new))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_keys_that_are_seen_and_not_finite(bad, d):
    """As in the formula: a score that is NaN or +inf makes its row NaN, one that is -inf has no weight.  Every place of a step's
    first 36 keys, in the first step and in a later one."""
    for at in [*range(36), *range(256, 292), 127, 511]:
        s = scores_case([0.0] * 600, d, new=2)
        s["k_cache"].view(-1, 2, d)[at, 0] = bad * s["q"][0, 0].sign()  # key/value head 0: of the query heads 0 and 1
        got = quest.paged_attention(**s)
        clean = scores_case([0.0] * at + [-1e4] + [0.0] * (599 - at), d, new=2)
        if bad == float("-inf"):
            check_attention(clean)
            same = (s["q"][:, :2].sign() == s["q"][0, 0].sign()).all(dim=-1)  # rows whose products all have one sign
            assert same[0, 0] and torch.isfinite(got[:, :2][same]).all()
        else:
            assert torch.isnan(got[0, 0]).all()
        assert torch.isfinite(got[:, 2:]).all()


def test_attention_pages_outside_the_pool_read_as_nothing():
    """A table entry that points nowhere is not read (keys and values 0), wherever it stands."""
    s = ref.paged_state(9, [64, 40], [1, 1], 2, 2, 64, 16)
    s["page_table"][0, 1], s["page_table"][1, 0] = 10 ** 6, -1
    got = quest.paged_attention(**s)
    k, v = s["k_cache"], s["v_cache"]
    zero = torch.zeros_like(k[:1])
    s["k_cache"], s["v_cache"] = torch.cat([k, zero]), torch.cat([v, zero])
    s["page_table"][0, 1] = s["page_table"][1, 0] = k.size(0)
    want, size = ref.attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"].cpu(), s["kv_lens"].tolist(), s["cu_new"].tolist(), 64 ** -0.5, s["q"])
    assert ((got.double().cpu() - want).abs() <= (2 ** -8 + 2 ** -10) * size + 2 ** -8 * want.abs() + 1e-30).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hq, hkv, kv, new", [(4, 2, 300, 200), (8, 1, 40, 5), (16, 16, 260, 260), (2, 1, 6000, 100), (8, 8, 5000, 3)])
def test_attention_later_tokens_that_are_not_finite_do_not_reach_earlier_rows(hq, hkv, kv, new, bad):
    """Keys and values of a chunk's later tokens, not finite in one column or in all: rows in front of them are as without, rows behind
    them are not finite where they have to be (a weight of zero times an infinity is a NaN in either)."""
    s = ref.paged_state(kv + new, [kv, 30], [new, 2], hq, hkv, 128 if new % 2 else 64, 16)
    clean = quest.paged_attention(**s).clone()
    first = kv - new // 2
    page = s["k_cache"].size(1)
    for j in range(first, kv):
        at = s["page_table"][0, j // page].long()
        s["v_cache"][at, j % page, :, 3 if j % 2 else slice(None)] = bad
        if j % 3 == 0:
            s["k_cache"][at, j % page, 0] = bad
    got = quest.paged_attention(**s)
    split = first - (kv - new)  # the chunk's rows in front of the first such token
    want, size = ref.attention(s["q"][:split], s["k_cache"], s["v_cache"], s["page_table"].cpu(), [first], [0, split], s["q"].size(2) ** -0.5, s["q"][:split])
    assert torch.isfinite(got[:split]).all() and torch.isfinite(got[new:]).all() and torch.equal(got[new:], clean[new:])
    assert ((got[:split].double().cpu() - want).abs() <= (2 ** -8 + 2 ** -10) * size + 2 ** -8 * want.abs() + 1e-30).all()
    assert not torch.isfinite(got[split:new, :, 3]).any()


def test_attention_is_the_same_call_after_call():
    s = ref.paged_state(10, [700, 3000, 90], [1, 40, 90], 16, 4, 128, 32)
    first = quest.paged_attention(**s).clone()
    for _ in range(5):
        assert torch.equal(quest.paged_attention(**s), first)


@pytest.mark.parametrize("seed", range(16))
def test_attention_random_batches(seed):
    """Batches of every kind of request over random heads and pages."""
    rng = random.Random(seed)
    hq, hkv = rng.choice([(1, 1), (8, 8), (6, 2), (16, 2), (40, 2), (65, 1), (128, 1), (100, 1), (24, 8)])
    batch = rng.randint(1, 9)
    kv = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 500)]) for _ in range(batch)]
    new = [rng.choice([0, min(n, 1), rng.randint(0, n), min(n, rng.randint(0, 9))]) for n in kv]
    if hq >= 64:
        new = [min(n, 30) for n in new]
    check_attention(ref.paged_state(100 + seed, kv, new, hq, hkv, rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 512, 1024]), pad=rng.choice([0, 5])))


@pytest.mark.parametrize("seed", range(8))
def test_attention_of_prompts_whose_tiles_are_cut_near_their_edges(seed):
    """From one to some ten places of the line per SM, in items of three to twelve places: cuts fall at, beside and into items."""
    rng = random.Random(seed)
    hq, hkv = rng.choice([(16, 16), (12, 12), (24, 8), (32, 4)])
    new = [rng.randint(100, 420) for _ in range(rng.randint(4, 9))]
    kv = [n + rng.choice([0, 0, rng.randint(1, 700)]) for n in new]
    check_attention(ref.paged_state(200 + seed, kv, new, hq, hkv, rng.choice([64, 128]), 64))


@pytest.mark.parametrize("hq, hkv, d, kv, new", [
    (8, 1, 128, [20000], [1]), (12, 2, 64, [9000, 3000], [4, 1]), (4, 4, 128, [4095], [1]), (5, 5, 64, [4097], [2]), (32, 1, 128, [6000, 1, 0, 40], [1, 1, 0, 3]),
    (1, 1, 64, [16385], [64]), (128, 1, 128, [8000], [1]), (8, 1, 128, [17000], [40]), (3, 1, 64, [16400, 700], [100, 300])])
def test_attention_of_few_long_items(hq, hkv, d, kv, new):
    """Items cut over hundreds of blocks, joined by a block per row or by eight rows a block, at one to three steps a piece."""
    check_attention(ref.paged_state(14 + hq, kv, new, hq, hkv, d, 64))


def test_attention_of_many_requests():
    """More requests than a block has threads: the sums take several rounds."""
    rng = random.Random(1)
    kv = [rng.choice([0, 1, 5, 17, 130]) for _ in range(900)]
    new = [min(n, rng.choice([0, 1, 1, 1, 3, 17])) for n in kv]
    check_attention(ref.paged_state(12, kv, new, 2, 1, 64, 16))


def test_attention_of_few_requests_among_very_many_without_rows():
    """The warp that lists the work walks over every request between two that have rows."""
    count = 150000
    kv, new = [0] * count, [0] * count
    for b, held, rows in ((0, 300, 1), (777, 140, 140), (90000, 17, 2), (count - 1, 600, 129)):
        kv[b], new[b] = held, rows
    check_attention(ref.paged_state(13, kv, new, 2, 2, 64, 64))


def test_attention_with_scale_zero_is_the_mean_of_what_is_seen():
    s = ref.paged_state(13, [150, 20], [30, 1], 2, 2, 64, 16)
    check_attention(s, scale=0.0)


def test_attention_lengths_beyond_the_table_and_offsets_beyond_the_rows_are_cut():
    s = ref.paged_state(14, [48, 30], [4, 2], 2, 2, 64, 16)  # three pages and a spare entry per request
    s["page_table"][0, 3] = s["page_table"][0, 2]
    s["kv_lens"][0] = 10 ** 9
    s["cu_new"][2] = 10 ** 6
    got = quest.paged_attention(**s)
    s["kv_lens"][0], s["cu_new"][2] = 64, 6
    # (the places behind the 48th token are NaN in this state: rows that see them are not finite in either)
    want = quest.paged_attention(**s)
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_attention_on_two_streams_at_once():
    states = [ref.paged_state(15 + i, [1500, 700, 60], [1, 90, 60], 8, 2, 128, 16) for i in range(2)]
    want = [quest.paged_attention(**s).clone() for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(quest.paged_attention(**states[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_attention_and_append_in_a_cache_with_more_than_2_31_elements():
    pages, page, hkv, d = 70000, 64, 4, 128
    k_cache, v_cache = (torch.empty(pages, page, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = ref.paged_state(17, [150, 70], [3, 70], 8, hkv, d, page)
    used = small["k_cache"].size(0)
    k_cache[-used:].copy_(small["k_cache"]), v_cache[-used:].copy_(small["v_cache"])
    want = quest.paged_attention(**small)
    table = torch.where(small["page_table"] >= 0, small["page_table"] + (pages - used), small["page_table"])
    assert torch.equal(quest.paged_attention(small["q"], k_cache, v_cache, table, small["kv_lens"], small["cu_new"]), want)
    qkv = torch.randn(2, (1 + 2 * hkv) * d, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([(pages - 1) * page + 63, (pages - 1) * page], device="cuda")
    quest.rope_paged_append(qkv, rope_table(d, 10).cuda(), i32([3, 4]), slots, k_cache, v_cache, 1)
    assert torch.equal(v_cache[-1, 63].flatten(), qkv[0, (1 + hkv) * d:]) and torch.equal(v_cache[-1, 0].flatten(), qkv[1, (1 + hkv) * d:])


def test_attention_waits_as_long_as_rows_in_front_of_a_nan_are_summed_again():
    """Eleven requests of 2^25 tokens over nine pages, two new tokens each, the second one's values NaN.  The first token's 32 rows are
    summed once more over up to 1.1 million keys by a warp, nearly three seconds in which the same stream's next item waits.  All scores
    are zero, so weights are one (some exponentials are off by 7.5e-5, the sums of 9743 steps in fp32 by at most 9743 * 2^-24; together
    below 2^-10), sums of values 0 and 1 are exact below 2^24, and a row is the mean of what it sees."""
    batch, page, d, heads, width = 11, 1024, 64, 32, 2 ** 15
    kv = width * page
    g = torch.Generator().manual_seed(0)
    v = torch.randint(0, 2, (9, page, 1, d), generator=g).bfloat16()
    v[8, -1] = float("nan")
    row = (torch.arange(width) % 8).int()
    row[-1] = 8
    q = torch.randn(2 * batch, heads, d, generator=g).bfloat16().cuda()
    table = row.expand(batch, width).contiguous().cuda()
    quest._lib.device_status()
    got = quest.paged_attention(q, torch.zeros_like(v).cuda(), v.cuda(), table, i32([kv] * batch), i32(list(range(0, 2 * batch + 1, 2))))
    got = got.double().cpu().view(batch, 2, heads, d)
    assert quest._lib.device_status() == 0
    sums = v.double()[:, :, 0].nan_to_num(0).sum(dim=1)
    want = (torch.bincount(row.long(), minlength=9).double() @ sums) / (kv - 1)
    assert ((got[:, 0] - want).abs() <= (2 ** -8 + 2 ** -10) * want).all()
    assert torch.isnan(got[:, 1]).all()


def test_attention_nothing_to_do():
    s = ref.paged_state(11, [5], [0], 4, 2, 64, 16)
    assert quest.paged_attention(**s).shape == (0, 4, 64)
    out = torch.full((3, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(out)
    quest.paged_attention(q, s["k_cache"], s["v_cache"], i32([]).view(0, 2), i32([]), i32([0]), out=out)
    assert (out == 5).all()


# ------------------------------------------------------------------------------------------------ drafted tokens
def drafts_case(seed, counts, vocab, dtype, noise=0.7):
    g = torch.Generator().manual_seed(seed)
    n, batch = sum(counts), len(counts)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    logits = 2 * torch.randn(n + batch, vocab, generator=g)
    rows = [cu[b] + b + i for b, c in enumerate(counts) for i in range(c)]
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[rows] + noise * torch.randn(n, vocab, generator=g), -1).to(dtype)
    tokens = torch.multinomial(draft.float(), 1, generator=g).view(-1) if n else torch.empty(0, dtype=torch.int64)
    return target, draft, tokens, cu, torch.rand(n + batch, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("counts, vocab, most", [
    ([0], 1, 0), ([1], 2, 1), ([3, 0, 5, 1], 97, 5), ([2] * 40, 1000, 2), ([8, 8, 0], 32000, 8), ([4, 4], 50257, 3), ([1, 2], 131072, 2), ([300], 40, 300)])
def test_verify_drafts(dtype, with_draft, counts, vocab, most):
    target, draft, tokens, cu, u = drafts_case(vocab + len(counts), counts, vocab, dtype)
    draft = draft if with_draft else None
    want, accepted = ref.verify(target, draft, tokens.tolist(), cu, u, most)
    got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), most, draft_probs=None if draft is None else draft.cuda())
    assert kept.tolist() == accepted and got.tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 8, 15, *range(2040, 2049)])
def test_verify_drafts_rows_of_any_alignment(vocab, dtype):
    """Rows and tensors that begin anywhere in 16 bytes, up to the last element of their memory, between entries that would be drawn."""
    target, draft, tokens, cu, u = drafts_case(vocab, [3, 0, 2, 4, 1] * 3, vocab, dtype)
    want, accepted = ref.verify(target, draft, tokens.tolist(), cu, u, 4)
    for offset in range(8):
        def placed(x):
            buffer = torch.full((offset + x.numel() + offset,), 1000.0, dtype=dtype, device="cuda")
            buffer[offset:offset + x.numel()] = x.cuda().view(-1)
            return buffer[offset:offset + x.numel()].view_as(x)
        got, kept = quest.verify_drafts(placed(target), tokens.cuda(), i32(cu), u.cuda(), 4, draft_probs=placed(draft))
        assert kept.tolist() == accepted and got.tolist() == want, offset


def test_verify_drafts_at_the_borders():
    """Equal distributions (nothing left to draw from when a draft is refused all the same), zero probabilities, uniforms of 0 and
    nearly 1, tokens outside the vocabulary, rows without any weight, NaN."""
    vocab = 600
    target = torch.zeros(12, vocab)
    target[:, 10], target[:, 300] = 0.25, 0.75
    draft = target[:6].clone()
    tokens = torch.tensor([10, 300, 11, -1, vocab, 10])
    cu = [0, 1, 2, 3, 4, 5, 6]
    last = 1 - 2.0 ** -24
    u = torch.tensor([0.5, 0.0, last, 0.25, 0.0, 0.0, 0.5, last, 0.0, 0.3, 0.1, 0.2])
    draft[0, 10] = 0.6                              # refused at u 0.5: 0.3 >= 0.25
    draft[5, 10], target[10, 10] = 0.25, 0.25       # kept
    target[11] = float("nan")
    want, accepted = ref.verify(target, draft, tokens.tolist(), cu, u, 1)
    got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), 1, draft_probs=draft.cuda())
    assert kept.tolist() == accepted and got.tolist() == want
    got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), 1)
    want, accepted = ref.verify(target, None, tokens.tolist(), cu, u, 1)
    assert kept.tolist() == accepted and got.tolist() == want


def test_verify_drafts_keeps_within_its_rows():
    """Offsets that run backwards or past the drafts are cut to what is there."""
    target, draft, tokens, cu, u = drafts_case(1, [2, 3], 50, torch.float32)
    got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32([0, 10 ** 6, -5]), u.cuda(), 3, draft_probs=draft.cuda())
    assert got.shape == (2, 4) and (kept >= 0).all() and (kept <= 3).all() and (got < 50).all()


def test_verify_drafts_follows_the_target():
    """Over many draws the first token is distributed as the target, whatever the draft: 20000 trials, five standard deviations."""
    trials, vocab = 20000, 5
    p, q = torch.tensor([0.5, 0.2, 0.15, 0.1, 0.05]), torch.tensor([0.1, 0.3, 0.2, 0.2, 0.2])
    g = torch.Generator().manual_seed(0)
    tokens = torch.multinomial(q, trials, replacement=True, generator=g)
    target, draft = p.expand(2 * trials, vocab).contiguous(), q.expand(trials, vocab).contiguous()
    got, _ = quest.verify_drafts(target.cuda(), tokens.cuda(), torch.arange(trials + 1, dtype=torch.int32, device="cuda"),
                                 torch.rand(2 * trials, generator=g).cuda(), 1, draft_probs=draft.cuda())
    share = torch.bincount(got[:, 0].cpu(), minlength=vocab) / trials
    assert ((share - p).abs() <= 5 * (p * (1 - p) / trials).sqrt()).all()


# ------------------------------------------------------------------------------------------------ streams, graphs
def test_serving_step_in_a_graph_follows_the_lengths():
    """Assign, append and attend captured once and replayed while the sequences grow, on a stream of its own."""
    hq, hkv, d, page, batch, width = 4, 2, 64, 16, 3, 8
    g = torch.Generator().manual_seed(1)
    table = rope_table(d, 200).cuda()
    k_cache, v_cache = (torch.full((batch * width, page, hkv, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    page_table, free_pages, free = torch.full((batch, width), -1, dtype=torch.int32, device="cuda"), torch.arange(batch * width, dtype=torch.int32, device="cuda"), i32([batch * width])
    lens, new = i32([0, 0, 0]), i32([0, 0, 0])
    rows = 40
    qkv = torch.zeros(rows, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device="cuda")

    def one_step():
        step = quest.page_assign(page_table, free_pages, free, lens, new, rows, page)
        q = quest.rope_paged_append(qkv, table, step.positions, step.slots, k_cache, v_cache, hq)
        quest.paged_attention(q, k_cache, v_cache, page_table, step.kv_lens, step.cu_new, out=out)
        lens.copy_(step.lens), free.copy_(step.free_count)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one_step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            one_step()
    torch.cuda.synchronize()
    history = [torch.zeros(0, (hq + 2 * hkv) * d, dtype=torch.bfloat16) for _ in range(batch)]
    for counts in ([17, 1, 20], [1, 1, 1], [16, 0, 3], [1, 30, 1]):
        x = torch.randn(rows, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16)
        qkv.copy_(x), new.copy_(i32(counts))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        row = 0
        for b, n in enumerate(counts):
            history[b] = torch.cat([history[b], x[row:row + n]])
            heads = history[b].view(-1, hq + 2 * hkv, d)
            cs = table.cpu()[:heads.size(0)]
            q, k, v = _rotate(heads[:, :hq], cs).double(), _rotate(heads[:, hq:hq + hkv], cs).double(), heads[:, hq + hkv:].double()
            for t in range(n):
                seen = heads.size(0) - n + t + 1
                s = torch.einsum("hgd,jhd->hgj", q[seen - 1].view(hkv, hq // hkv, d), k[:seen]) * d ** -0.5
                p = torch.softmax(s, -1)
                want, size = torch.einsum("hgj,jhd->hgd", p, v[:seen]).reshape(hq, d), torch.einsum("hgj,jhd->hgd", p, v[:seen].abs()).reshape(hq, d)
                error = (out[row + t].double().cpu() - want).abs()
                assert (error <= (2 ** -8 + 2 ** -10) * size + 2 ** -8 * want.abs()).all()
            row += n
    assert lens.tolist() == [h.size(0) for h in history]


_BATCHES_OF_A_NEW_PROCESS = """
import torch
import quest_b200 as quest

i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
for batch in range(6116, 6150):  # shared memory goes from below to beyond what a launch has without asking, the kernels' own variables included
    table, free = torch.full((batch, 1), -1, dtype=torch.int32, device="cuda"), torch.arange(batch, dtype=torch.int32, device="cuda")
    zeros, ones = torch.zeros(batch, dtype=torch.int32, device="cuda"), torch.ones(batch, dtype=torch.int32, device="cuda")
    step = quest.page_assign(table, free, i32([batch]), zeros, ones, batch, 16)
    assert step.free_count.tolist() == [0] and torch.equal(step.kv_lens, ones) and torch.equal(table[:, 0], free.flip(0)), batch
    assert torch.equal(step.slots, 16 * free.flip(0).long()), batch
    left = quest.page_release(table, free, step.free_count, step.lens, zeros, 16)
    assert left.tolist() == [batch] and torch.equal(free, table[:, 0]), batch
print("every batch was served")
"""


def test_page_tables_of_batches_that_just_need_more_shared_memory():
    """In a process that has asked for nothing larger before, ascending."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(quest.__file__)))
    run = subprocess.run([sys.executable, "-c", _BATCHES_OF_A_NEW_PROCESS], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "every batch was served" in run.stdout, run.stderr[-2000:]


def test_page_tables_of_two_threads_with_different_batches():
    """The shared memory that one call asks for does not shrink what another call's launch has."""
    failures = []

    def work(batch):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                table, free = torch.zeros(batch, 1, dtype=torch.int32, device="cuda"), torch.arange(batch, dtype=torch.int32, device="cuda")
                zeros, ones, count = torch.zeros_like(free), torch.ones_like(free), i32([batch])
                for _ in range(400):
                    step = quest.page_assign(table, free, count, zeros, ones, batch, 16)
                    quest.page_release(table, free.clone(), step.free_count, step.lens, zeros, 16)
                assert step.free_count.item() == 0
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(batch,)) for batch in (8192, 6200, 7000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [97, 2048])
def test_verify_drafts_with_probabilities_that_are_none(vocab, dtype):
    """Negative probabilities count as 0 on both sides.  A draft whose own probability is NaN is refused, and where a draft's probability
    is NaN nothing is drawn in its place."""
    target, draft, tokens, cu, u = drafts_case(vocab, [4, 2, 0, 3, 1] * 8, vocab, dtype)
    g = torch.Generator().manual_seed(vocab)
    n = tokens.numel()
    below = torch.rand(draft.shape, generator=g) < 0.3
    below[torch.arange(n), tokens] = torch.rand(n, generator=g) < 0.3  # the drafted token's among them
    draft = torch.where(below, -3 * draft - 0.25, draft)
    target = torch.where(torch.rand(target.shape, generator=g) < 0.2, -target - 0.125, target)

    def check(draft):
        want, accepted = ref.verify(target.clamp(min=0), draft.clamp(min=0), tokens.tolist(), cu, u, 4)  # clamp leaves a NaN
        got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), 4, draft_probs=draft.cuda())
        assert kept.tolist() == accepted and got.tolist() == want

    check(draft)
    none = torch.rand(draft.shape, generator=g) < 0.2
    none[torch.arange(n), tokens] = torch.rand(n, generator=g) < 0.3
    check(torch.where(none, float("nan"), draft))
    # nothing of the target's mass lies where a draft was below zero: what is drawn there is the target's own row
    p = torch.tensor([[0.0, 0.0, 0.25, 0.75], [0.25] * 4]).to(dtype).cuda()
    q = torch.tensor([[0.5, -4.0, 0.5, 0.0]]).to(dtype).cuda()
    got, kept = quest.verify_drafts(p, torch.tensor([1], device="cuda"), i32([0, 1]), torch.tensor([0.5, 0.0], device="cuda"), 1, draft_probs=q)
    assert kept.tolist() == [0] and got.tolist() == [[3, -1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["whole", "half", "tiny", "peak", "large"])
@pytest.mark.parametrize("vocab, batch", [(40, 200), (138, 200), (5003, 100), (131072, 24)])
def test_verify_drafts_next_to_the_borders(vocab, batch, kind, dtype):
    """Uniforms that fall as near to a border between two tokens as fp32 can: the token is that of the sums in 64 bits, whatever is left
    of a row (a millionth of it, or weights that are no probabilities) and however far apart the sizes of its weights are."""
    g = torch.Generator().manual_seed(vocab + len(kind))
    logits = 1.5 * torch.randn(batch, vocab, generator=g, dtype=torch.float64)
    p = torch.softmax(logits, -1)
    noise = torch.randn(batch, vocab, generator=g, dtype=torch.float64)
    q = torch.softmax(logits + {"tiny": 1e-6 if dtype is torch.float32 else 1e-4}.get(kind, 0.7) * noise, -1)
    if kind == "peak":
        at = torch.randint(0, vocab, (batch, 1), generator=g)
        p, q = (0.4 * p).scatter(1, at, 0.6), q.scatter(1, at, 1.3e-6)
    p, q = (p * (1000 if kind == "large" else 1)).to(dtype), (q * (1000 if kind == "large" else 1)).to(dtype)
    counts = [0 if kind == "whole" else 1] * batch
    target = p if kind == "whole" else torch.stack([p, p], 1).flatten(0, 1)
    draft = None if kind == "whole" else q
    tokens = torch.empty(0, dtype=torch.int64) if draft is None else (q.double() / p.double().clamp(min=1e-300)).argmax(1)
    cu = [sum(counts[:b]) for b in range(batch + 1)]
    u = torch.zeros(target.size(0))
    for b in range(batch):
        w = p[b].double() if draft is None else (p[b].double() - q[b].double()).clamp(min=0)
        if w.sum() == 0:  # (all refused drafts of a small vocabulary in bf16: the same rows)
            w = p[b].double()
        sums = w.cumsum(0)
        border = sums[torch.randint(0, vocab, (1,), generator=g).item()] / sums[-1]
        u[cu[b] + b + counts[b]] = border.float().clamp(max=1 - 2.0 ** -24)
        if counts[b]:
            u[cu[b] + b] = 1 - 2.0 ** -24  # refuses where q is more than p
    want, accepted = ref.verify(target, draft, tokens.tolist(), cu, u, 1)
    got, kept = quest.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), 1, draft_probs=None if draft is None else draft.cuda())
    assert kept.tolist() == accepted
    assert got.tolist() == want, [(b, x, y) for b, (x, y) in enumerate(zip(got.tolist(), want)) if x != y][:5]
    if kind != "tiny":
        assert sum(accepted) < batch // 8 + 1
