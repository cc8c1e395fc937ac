"""The decoder over a paged cache: against its own forward pass over whole sequences, and the loops around it."""
from __future__ import annotations

import pytest
import torch

from quest_b200 import serving
from quest_b200.prefill import Decoder, DecoderConfig, swap_linears

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(n_embd=512, n_layer=2, n_head=4, ffn=768, vocab_size=300, sequence_length=256)


def make_model(mode, seed=0):
    with torch.random.fork_rng(devices=[0]):
        torch.manual_seed(seed)
        with torch.device("cuda"):
            model = Decoder(CFG).to(torch.bfloat16).eval()
            for p in model.parameters():  # livelier than the initialisation for training, so that attention matters
                if p.dim() > 1:
                    p.data.mul_(3)
    return swap_linears(model, mode) if mode != "bf16" else model


def prompts_of(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG.vocab_size, (n,), generator=g) for n in lengths]


def relative(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("page_size", [16, 64])
def test_paged_forward_equals_the_forward_of_whole_sequences(page_size):
    """bf16 linears: both passes round at the same places but for the attention (its probabilities to bf16) and the rotary
    embedding; each bf16 rounding is 2^-9 of a value on average, and two layers have about ten of them in line."""
    model = make_model("bf16")
    prompts = prompts_of([1, 17, 128, 200])
    cache = serving.PagedCache(CFG, 64, 5, page_size=page_size)
    new = torch.tensor([p.numel() for p in prompts] + [0], dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        hidden, step = serving.extend(model, cache, torch.cat(prompts).cuda(), new)
        whole = [model(p.cuda()[None])[0] for p in prompts]
    assert step.kv_lens.tolist() == [1, 17, 128, 200, 0] and cache.lens.tolist() == [1, 17, 128, 200, 0]
    for b, w in enumerate(whole):
        assert relative(hidden[step.cu_new[b]:step.cu_new[b + 1]], w) < 10 * 2 ** -9


@pytest.mark.parametrize("mode", ["bf16", "int4", "int4_fused"])
def test_chunks_and_single_tokens_equal_one_pass_over_the_cache(mode):
    """The same tokens in one step, or as chunks and single tokens: rows of the linears do not depend on one another, the attention
    sums in another order.  With int4 activations a value at a border can change its code, so only the bulk is compared."""
    model = make_model(mode)
    prompts = prompts_of([90, 33])
    whole = serving.PagedCache(CFG, 16, 2, page_size=16)
    new = torch.tensor([90, 33], dtype=torch.int32, device="cuda")
    hidden, step = serving.extend(model, whole, torch.cat(prompts).cuda(), new)
    parts = serving.PagedCache(CFG, 16, 2, page_size=16)
    got = [[], []]
    at = [0, 0]
    for counts in ([50, 1], [1, 20], [38, 0], [1, 12]):
        x = torch.cat([p[a:a + c] for p, a, c in zip(prompts, at, counts)]).cuda()
        h, s = serving.extend(model, parts, x, torch.tensor(counts, dtype=torch.int32, device="cuda"))
        for b in range(2):
            got[b].append(h[s.cu_new[b]:s.cu_new[b + 1]])
            at[b] += counts[b]
    assert parts.lens.tolist() == [90, 33] == whole.lens.tolist() and parts.free_count.item() == whole.free_count.item()
    for b in range(2):
        a, w = torch.cat(got[b]), hidden[step.cu_new[b]:step.cu_new[b + 1]]
        assert relative(a, w) < (10 * 2 ** -9 if mode == "bf16" else 0.35)


@pytest.mark.parametrize("mode", ["bf16", "int4_fused"])
def test_padding_rows_are_zero_and_change_nothing(mode):
    model = make_model(mode)
    prompt = prompts_of([40])[0].cuda()
    new = torch.tensor([40, 0], dtype=torch.int32, device="cuda")
    a, _ = serving.extend(model, serving.PagedCache(CFG, 8, 2, page_size=16), prompt, new)
    b, _ = serving.extend(model, serving.PagedCache(CFG, 8, 2, page_size=16), torch.cat([prompt, prompt[:9]]), new)
    assert torch.isfinite(b).all()
    if mode == "bf16":
        assert relative(b[:40], a) < 10 * 2 ** -9


def test_generate_equals_the_loop_without_a_cache():
    """Greedy tokens of the same model by whole forward passes; where its two best logits are closer than the rounding of bf16
    may move them, the sequence may part, so each step's choice is compared under the tokens chosen by generate."""
    model = make_model("bf16")
    prompts = prompts_of([3, 30, 64])
    cache = serving.PagedCache(CFG, 24, 4, page_size=16)
    got = serving.generate(model, cache, prompts, 20)
    assert got.shape == (3, 20) and cache.free_count.item() == 24 and cache.lens.tolist() == [0] * 4
    with torch.inference_mode():
        for b, p in enumerate(prompts):
            sequence = torch.cat([p.cuda(), got[b]])
            logits = model.lm_head(model(sequence[None])[0]).float()[p.numel() - 1:-1]
            chosen = logits.gather(1, got[b][:, None])[:, 0]
            assert (logits.amax(dim=1) - chosen <= 20 * 2 ** -9 * logits.abs().amax(dim=1)).all()
    again = serving.generate(model, cache, prompts, 20)  # pages are used again, in another order
    assert torch.equal(again, got)


def test_generate_refuses_what_does_not_fit():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 4, 2, page_size=16)
    with pytest.raises(ValueError):
        serving.generate(model, cache, prompts_of([1, 1, 1]), 1)
    with pytest.raises(ValueError):
        serving.generate(model, cache, prompts_of([40, 40]), 1)
    with pytest.raises(ValueError):
        serving.generate(model, cache, [torch.empty(0, dtype=torch.long)], 1)
    with pytest.raises(AssertionError):
        serving.PagedCache(CFG, 4, 2, max_length=257)


def test_decoding_step_in_a_graph():
    """A captured step replayed token after token gives what eager steps give."""
    model = make_model("int4_fused")
    prompts = prompts_of([20, 35])
    new = torch.tensor([20, 35], dtype=torch.int32, device="cuda")
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    tokens = prompts_of([2], seed=5)[0].cuda()
    feed = [prompts_of([2], seed=s)[0].cuda() for s in range(6, 12)]

    def run(graphed):
        cache = serving.PagedCache(CFG, 16, 2, page_size=16)
        serving.extend(model, cache, torch.cat(prompts).cuda(), new)
        held = torch.empty_like(tokens)
        if graphed:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            state = [t.clone() for t in (cache.lens, cache.free_count, cache.page_table)]
            with torch.cuda.stream(side):
                held.copy_(tokens)
                serving.extend(model, cache, held, one)
            torch.cuda.current_stream().wait_stream(side)
            for t, x in zip((cache.lens, cache.free_count, cache.page_table), state):
                t.copy_(x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                hidden, _ = serving.extend(model, cache, held, one)
        out = []
        for x in feed:
            held.copy_(x)
            if graphed:
                graph.replay()
                out.append(hidden.clone())
            else:
                out.append(serving.extend(model, cache, held, one)[0])
        return torch.stack(out), cache.lens.tolist()

    eager, lens = run(False)
    graphed, lens_g = run(True)
    assert lens == lens_g == [26, 41] and torch.equal(eager, graphed)


@pytest.mark.parametrize("count", [0, 1, 4])
def test_verify_takes_refused_drafts_out_again(count):
    """Drafts that are the target's own greedy tokens under a sharpened model are kept, others refused; the cache afterwards holds
    exactly the kept ones, whatever was written.  Which of two tokens leads is settled only where their logits are further apart than
    the roundings of bf16 may move them, the bound of the test of generate: the second request's first two candidates behind its first
    draft have the logits 624 and 620 (bf16 has a step of 4 there, and ten roundings of 2^-9 in line make 12), and a tie halves the
    probability, which u = 0.5 refuses.  Drafts within that bound may be kept or not."""
    model = make_model("bf16")
    model.lm_head.weight.data.mul_(200)  # nearly all probability on one token
    prompts = prompts_of([10, 25])
    cache = serving.PagedCache(CFG, 16, 2, page_size=16)
    serving.extend(model, cache, torch.cat(prompts).cuda(), torch.tensor([10, 25], dtype=torch.int32, device="cuda"))
    reference = serving.PagedCache(CFG, 16, 2, page_size=16)
    last = torch.tensor([7, 11], device="cuda")
    chain = serving.generate(model, reference, [torch.cat([p, t.cpu()[None]]) for p, t in zip(prompts, last)], max(count, 1))
    drafts = chain[:, :count].clone()
    if count:
        drafts[1, count // 2] = (drafts[1, count // 2] + 1) % CFG.vocab_size  # the second request's drafts go wrong there
    u = torch.full((2, count + 1), 0.5, device="cuda")
    free = cache.free_count.item()
    tokens, kept = serving.verify(model, cache, last, drafts, u)
    for b, p in enumerate(prompts):
        with torch.inference_mode():
            logits = model.lm_head(model(torch.cat([p.cuda(), last[b:b + 1], drafts[b]])[None])[0]).float()[p.numel():]
        noise = 20 * 2 ** -9 * logits.abs().amax(dim=1)
        own = logits[:-1].gather(1, drafts[b][:, None])[:, 0]
        lead = own - logits[:-1].scatter(1, drafts[b][:, None], float("-inf")).amax(dim=1)  # over the best other token
        surely_kept, surely_refused = (lead > noise[:-1]).tolist() + [False], (lead < -noise[:-1]).tolist() + [True]
        k = kept[b].item()
        assert surely_kept.index(False) <= k <= surely_refused.index(True)
        assert tokens[b, :k].tolist() == drafts[b, :k].tolist() and (tokens[b, k + 1:] == -1).all()
        if k == count or lead[k] < -noise[k]:  # drawn from nearly one token
            assert logits[k].max() - logits[k, tokens[b, k]] <= noise[k]
    if count:
        assert kept[1].item() <= count // 2
    assert cache.lens.tolist() == [10 + 1 + kept[0].item(), 25 + 1 + kept[1].item()]
    held = sum(-(-n // 16) for n in cache.lens.tolist())
    assert cache.free_count.item() == 16 - held and free >= cache.free_count.item()
    assert sorted(cache.free_pages[:16 - held].tolist() + cache.page_table[0, :-(-cache.lens[0].item() // 16)].tolist()
                  + cache.page_table[1, :-(-cache.lens[1].item() // 16)].tolist()) == list(range(16))
    # the next step attends over the kept tokens: the same as a cache that never saw the refused ones
    clean = serving.PagedCache(CFG, 16, 2, page_size=16)
    sequences = [torch.cat([p.cuda(), last[b:b + 1], drafts[b, :kept[b]]]) for b, p in enumerate(prompts)]
    serving.extend(model, clean, torch.cat(sequences), torch.tensor([s.numel() for s in sequences], dtype=torch.int32, device="cuda"))
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    a, _ = serving.extend(model, cache, last, one)
    b, _ = serving.extend(model, clean, last, one)
    assert relative(a, b) < 10 * 2 ** -9


def test_requests_without_pages_are_refused_and_recover():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 3, 2, page_size=16)
    _, step = serving.extend(model, cache, prompts_of([60])[0].cuda(), torch.tensor([30, 30], dtype=torch.int32, device="cuda"))
    assert step.kv_lens.tolist() == [30, 0] and cache.lens.tolist() == [30, 0] and cache.free_count.item() == 1
    cache.shorten(torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert cache.free_count.item() == 3
    _, step = serving.extend(model, cache, prompts_of([30])[0].cuda(), torch.tensor([0, 30], dtype=torch.int32, device="cuda"))
    assert step.kv_lens.tolist() == [0, 30]


def test_verify_leaves_places_that_are_not_active():
    """With u = 0 a draft of the vocabulary is kept and the first token drawn, whatever the logits round to; a draft outside it is
    refused.  The cache afterwards is one that took the active places' tokens alone."""
    model = make_model("bf16")
    prompts, count = prompts_of([10, 20, 25]), 3
    cache, alone = (serving.PagedCache(CFG, 16, n, page_size=16) for n in (4, 2))
    i32 = dict(dtype=torch.int32, device="cuda")
    serving.extend(model, cache, torch.cat(prompts).cuda(), torch.tensor([10, 20, 0, 25], **i32))
    serving.extend(model, alone, torch.cat([prompts[0], prompts[2]]).cuda(), torch.tensor([10, 25], **i32))
    last = torch.tensor([7, 400, -1, 11], device="cuda")  # what stands at the other places is never looked up
    drafts = torch.tensor([[5, 6, 7], [8, 9, 10], [10 ** 6] * 3, [11, 10 ** 6, 12]], device="cuda")
    drafts[3, 1:] %= CFG.vocab_size
    q = torch.zeros(4, count, CFG.vocab_size, device="cuda")
    q[3, 1, drafts[3, 1]] = float("nan")  # u q is then not below p: refused
    active = torch.tensor([True, False, False, True], device="cuda")
    tokens, kept = serving.verify(model, cache, last, drafts, torch.zeros(4, count + 1, device="cuda"), draft_probs=q, active=active)
    assert kept.tolist() == [3, 0, 0, 1] and tokens.tolist() == [[5, 6, 7, 0], [-1] * 4, [-1] * 4, [11, 0, -1, -1]]
    assert cache.lens.tolist() == [14, 20, 0, 27] and cache.free_count.item() == 16 - (1 + 2 + 0 + 2)
    new = torch.tensor([4, 2], **i32)
    serving.extend(model, alone, torch.tensor([7, 5, 6, 7, 11, 11], device="cuda"), new)
    a, _ = serving.extend(model, cache, torch.tensor([1, 2, 3], device="cuda"), torch.tensor([1, 1, 0, 1], **i32))
    b, _ = serving.extend(model, alone, torch.tensor([1, 3], device="cuda"), torch.tensor([1, 1], **i32))
    assert relative(a[[0, 2]], b) < 10 * 2 ** -9


def test_verify_answers_nothing_for_a_request_without_pages():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 3, 2, page_size=16)
    serving.extend(model, cache, prompts_of([46])[0].cuda(), torch.tensor([30, 16], dtype=torch.int32, device="cuda"))
    drafts = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    tokens, kept = serving.verify(model, cache, torch.tensor([1, 2], device="cuda"), drafts, torch.full((2, 2), 0.5, device="cuda"))
    assert tokens[0, 0].item() >= 0 and tokens[1].tolist() == [-1, -1] and kept[1].item() == 0
    assert cache.lens.tolist() == [31 + kept[0].item(), 16] and cache.free_count.item() == 0


def test_generate_counts_the_pages_that_are_free():
    """Pages that another place holds are not there for new prompts; the last new token needs no room."""
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 3, 2, page_size=16)
    held = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    serving.extend(model, cache, prompts_of([20])[0].cuda(), held)
    with pytest.raises(ValueError):
        serving.generate(model, cache, prompts_of([10]), 8)
    assert serving.generate(model, cache, prompts_of([10]), 7).shape == (1, 7)
    assert cache.lens.tolist() == [0, 20] and cache.free_count.item() == 1
    assert serving.generate(model, cache, [], 4).shape == (0, 4)


def test_shorten_takes_negative_lengths_for_zero():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 4, 2, page_size=16)
    serving.extend(model, cache, prompts_of([40])[0].cuda(), torch.tensor([20, 20], dtype=torch.int32, device="cuda"))
    cache.shorten(torch.tensor([-5, 100], dtype=torch.int32, device="cuda"))
    assert cache.lens.tolist() == [0, 20] and cache.free_count.item() == 2


@pytest.mark.parametrize("max_length", [100, 33, 9])
def test_requests_grow_to_the_cache_length_whatever_the_page_size(max_length):
    """A length that is not whole pages: the last page is used up to it, and not beyond."""
    model = make_model("bf16")
    page = 16
    cache = serving.PagedCache(CFG, 24, 3, max_length=max_length, page_size=page)
    i32 = dict(dtype=torch.int32, device="cuda")
    prompt = prompts_of([max_length])[0].cuda()
    hidden, step = serving.extend(model, cache, prompt, torch.tensor([max_length, 0, 0], **i32))
    assert step.kv_lens.tolist() == [max_length, 0, 0] == cache.lens.tolist() and cache.free_count.item() == 24 - -(-max_length // page)
    with torch.inference_mode():
        assert relative(hidden, model(prompt[None])[0]) < 10 * 2 ** -9
    # one token more is refused, what lies behind it in the batch is served, and what the step says is what the cache holds
    free = cache.free_count.item()
    for new in ([1, 3, max_length], [2 ** 31 - 1, 0, 0], [5, 0, 1]):
        before = cache.lens.tolist()
        rows = sum(min(n, 2 * max_length) for n in new)
        _, step = serving.extend(model, cache, torch.zeros(rows, dtype=torch.long, device="cuda"), torch.tensor(new, **i32))
        # (where the rows end within a request those behind it are refused, too: the second batch's)
        served = [held + n <= max_length and sum(new[:b + 1]) <= rows for b, (held, n) in enumerate(zip(before, new))]
        held = [b + n if s else b for b, n, s in zip(before, new, served)]
        assert cache.lens.tolist() == held == step.lens.tolist()
        assert step.kv_lens.tolist() == [h if s else 0 for h, s in zip(held, served)]
        assert cache.free_count.item() == 24 - sum(-(-h // page) for h in held)
        slots = step.slots.tolist()
        assert all(s == -1 for s in slots[:min(new[0], rows)])
    # a step of fewer new tokens is granted as always, negative ones count as none
    _, step = serving.extend(model, cache, torch.zeros(2, dtype=torch.long, device="cuda"), torch.tensor([-7, 2, 0], **i32))
    assert step.kv_lens.tolist() == [max_length, 5, max_length]
    cache.shorten(torch.zeros(3, **i32))
    assert cache.free_count.item() == 24 and free <= 24
    tokens = serving.generate(model, cache, [prompt[:4].cpu()], max_length - 3)  # the last one is not kept
    assert tokens.shape == (1, max_length - 3) and cache.free_count.item() == 24
    with pytest.raises(ValueError, match="length"):
        serving.generate(model, cache, [prompt[:4].cpu()], max_length - 2)


def test_verify_at_the_cache_length():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 24, 2, max_length=40, page_size=16)
    i32 = dict(dtype=torch.int32, device="cuda")
    serving.extend(model, cache, prompts_of([70])[0].cuda(), torch.tensor([38, 32], **i32))
    drafts, u = torch.zeros(2, 2, dtype=torch.long, device="cuda"), torch.zeros(2, 3, device="cuda")
    tokens, kept = serving.verify(model, cache, torch.tensor([1, 2], device="cuda"), drafts, u)  # 38 + 3 do not fit, 32 + 3 do
    assert tokens[0].tolist() == [-1] * 3 and kept.tolist() == [0, 2] and cache.lens.tolist() == [38, 35]
    assert cache.free_count.item() == 24 - 3 - 3


def test_verify_without_drafts_but_with_their_probabilities():
    model = make_model("bf16")
    cache, other = (serving.PagedCache(CFG, 16, 2, page_size=16) for _ in range(2))
    for c in (cache, other):
        serving.extend(model, c, prompts_of([30])[0].cuda(), torch.tensor([10, 20], dtype=torch.int32, device="cuda"))
    last, drafts, u = torch.tensor([7, 11], device="cuda"), torch.empty(2, 0, dtype=torch.long, device="cuda"), torch.tensor([[0.2], [0.7]], device="cuda")
    want, _ = serving.verify(model, other, last, drafts, u)
    got, kept = serving.verify(model, cache, last, drafts, u, draft_probs=torch.empty(2, 0, CFG.vocab_size, device="cuda"))
    assert got.tolist() == want.tolist() and got.shape == (2, 1) and kept.tolist() == [0, 0] and cache.lens.tolist() == [11, 21]


def test_verify_refuses_before_the_cache_changes():
    model = make_model("bf16")
    cache = serving.PagedCache(CFG, 16, 2, page_size=16)
    serving.extend(model, cache, prompts_of([30])[0].cuda(), torch.tensor([10, 20], dtype=torch.int32, device="cuda"))
    good = dict(tokens=torch.tensor([7, 11], device="cuda"), drafts=torch.zeros(2, 3, dtype=torch.long, device="cuda"), uniforms=torch.zeros(2, 4, device="cuda"),
                draft_probs=torch.zeros(2, 3, CFG.vocab_size, device="cuda"), active=torch.tensor([True, False], device="cuda"))
    table = cache.page_table.clone()
    for name, bad in (("tokens", torch.zeros(3, dtype=torch.long, device="cuda")), ("drafts", torch.zeros(3, 3, dtype=torch.long, device="cuda")),
                      ("drafts", torch.zeros(2, 3, dtype=torch.int32, device="cuda")), ("drafts", torch.zeros(2, dtype=torch.long, device="cuda")),
                      ("uniforms", torch.zeros(2, 3, device="cuda")), ("uniforms", torch.zeros(2, 4, dtype=torch.float64, device="cuda")),
                      ("uniforms", torch.zeros(2, 4)), ("draft_probs", torch.zeros(2, 3, CFG.vocab_size + 1, device="cuda")),
                      ("draft_probs", torch.zeros(2, 3, CFG.vocab_size, dtype=torch.bfloat16, device="cuda")),
                      ("active", torch.ones(2, dtype=torch.int32, device="cuda")), ("active", torch.ones(3, dtype=torch.bool, device="cuda"))):
        with pytest.raises(ValueError):
            serving.verify(model, cache, **{**good, name: bad})
        assert cache.lens.tolist() == [10, 20] and cache.free_count.item() == 13 and torch.equal(cache.page_table, table)
    assert serving.verify(model, cache, **good)[1].tolist() == [3, 0] and cache.lens.tolist() == [14, 20]


@pytest.mark.parametrize("mode", ["bf16", "int4_fused"])
def test_pages_refuse_where_a_gradient_is_asked_for(mode):
    """The attention over pages leaves no graph: outside no_grad its part of a gradient would be missing without a word."""
    model = make_model("bf16")
    prompt = prompts_of([20])[0].cuda()
    cache = serving.PagedCache(CFG, 8, 1, page_size=16)
    step = cache.assign(torch.tensor([20], dtype=torch.int32, device="cuda"), 20)
    with pytest.raises(RuntimeError, match="gradient"):
        model(prompt[None], cache.layers(step))
    assert not any(k.any() for k in cache.k)  # before anything is written
    if mode != "bf16":
        model = swap_linears(model, mode)
    with torch.no_grad():
        a = model(prompt[None], cache.layers(step))[0]
    with torch.inference_mode():
        b = model(prompt[None], cache.layers(step))[0]
    assert torch.equal(a, b)


class Follows(torch.nn.Module):
    """A model whose next token is a function of the last one alone, with all of the probability on it."""

    def __init__(self, successor):
        super().__init__()
        vocab = len(successor)
        self.lm_head = torch.nn.Linear(vocab, vocab, bias=False, device="cuda")
        self.lm_head.weight.data.zero_()
        self.lm_head.weight.data[successor, torch.arange(vocab)] = 1e4

    def forward(self, idx, pages):
        return torch.nn.functional.one_hot(idx, self.lm_head.in_features).float()


@pytest.mark.parametrize("count", [0, 1, 3])
def test_verify_reads_every_active_place_its_own_logits(count):
    """Every subset of four places: drafts are kept as far as they follow, the next token is what follows the last kept one, whichever
    rows the places' tokens have in the packed batch."""
    vocab, places = 50, 4
    g = torch.Generator().manual_seed(count)
    successor = torch.randperm(vocab, generator=g)
    model = Follows(successor)
    for subset in [None, *range(16)]:
        cache = serving.PagedCache(CFG, 16, places, page_size=16)
        cache.assign(torch.tensor([3, 20, 0, 15], dtype=torch.int32, device="cuda"), 38)
        active = None if subset is None else [bool(subset >> b & 1) for b in range(places)]
        last = torch.randint(0, vocab, (places,), generator=g)
        drafts, right = torch.empty(places, count, dtype=torch.long), []
        for b in range(places):
            follows = int(torch.randint(0, count + 1, (1,), generator=g))
            token = last[b]
            for i in range(count):
                token = successor[token] if i != follows else (successor[token] + 1) % vocab
                drafts[b, i] = token
            right.append(follows)
        want, kept = [], []
        for b in range(places):
            if active is not None and not active[b]:
                want.append([-1] * (count + 1)), kept.append(0)
                last[b], drafts[b] = (-1, 10 ** 6)[b % 2], 10 ** 6  # never looked up
            else:
                sequence = [int(last[b]), *drafts[b, :right[b]].tolist()]
                want.append(sequence[1:] + [int(successor[sequence[-1]])] + [-1] * (count - right[b])), kept.append(right[b])
        u = torch.rand(places, count + 1, generator=g)
        got, accepted = serving.verify(model, cache, last.cuda(), drafts.cuda(), u.cuda(), active=None if active is None else torch.tensor(active, device="cuda"))
        assert got.tolist() == want and accepted.tolist() == kept
        assert cache.lens.tolist() == [n + (0 if active is not None and not active[b] else 1 + kept[b]) for b, n in enumerate([3, 20, 0, 15])]


def test_captured_steps_run_up_to_the_cache_length_and_verify():
    """A step of single tokens and a speculative step, captured over a cache whose length is not whole pages, replayed past its end."""
    vocab, count = 50, 2
    successor = torch.randperm(vocab, generator=torch.Generator().manual_seed(1))
    model = Follows(successor)
    i32 = dict(dtype=torch.int32, device="cuda")

    def run(graphed):
        cache = serving.PagedCache(CFG, 16, 2, max_length=39, page_size=16)
        cache.assign(torch.tensor([30, 31], **i32), 61)
        state = [t.clone() for t in (cache.lens, cache.free_count, cache.page_table, cache.free_pages)]
        one, last = torch.ones(2, **i32), torch.tensor([3, 4], device="cuda")
        drafts, u, active = torch.zeros(2, count, dtype=torch.long, device="cuda"), torch.full((2, count + 1), 0.5, device="cuda"), torch.tensor([True, False], device="cuda")

        def step():
            tokens, kept = serving.verify(model, cache, last, drafts, u, active=active)
            _, single = serving.extend(model, cache, last, one)
            return tokens, kept, single.kv_lens, single.slots, cache.lens.clone(), cache.free_count.clone()

        if graphed:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            for t, x in zip((cache.lens, cache.free_count, cache.page_table, cache.free_pages), state):
                t.copy_(x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                results = step()
        out = []
        for i in range(8):
            last.copy_(torch.tensor([3 + i, 4]))
            first = int(successor[3 + i])
            drafts[0] = torch.tensor([first, int(successor[first]) if i % 2 else 0])
            active.copy_(torch.tensor([True, i > 4]))
            if graphed:
                graph.replay()
            out.append([x.tolist() for x in (results if graphed else step())])
        return out

    eager = run(False)
    assert run(True) == eager
    assert eager[-1][4] == [39, 39] and eager[-1][0] == [[-1] * 3] * 2 and eager[-1][2] == [0, 0]  # by then both are full
