"""Sampling decode from the 4-bit cache: branches, drafts, retrieval and page moves end to end."""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from popkv_b200.decoder import LlamaConfig, LlamaWeights
from popkv_b200.kv4_decode import Kv4Decoder, main
from popkv_b200.popkv import RetrievalConfig

pytestmark = pytest.mark.gpu

CONFIG = LlamaConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512,
                     vocab_size=503, num_hidden_layers=3)


@pytest.fixture(scope="module")
def weights(cuda_device):
    return LlamaWeights.random(CONFIG, device=cuda_device, std=0.06, seed=3)


def prompt(tokens, seed=0):
    return torch.randint(0, CONFIG.vocab_size, (tokens,), generator=torch.Generator().manual_seed(seed))


def near(a, b):
    """Logits of the same tokens by another route: the routes differ by bf16 roundings (2^-8 of a value) in 3
    layers and the head, each of which moves a logit by at most a few of its own; 12 of them of the spread."""
    return float((a - b).abs().max()) <= 12 * 2.0 ** -8 * float(b.std() + b.abs().max())


def test_several_tokens_in_one_pass_are_the_single_steps(weights, cuda_device):
    one, many = (Kv4Decoder(weights, max_seqs=2, max_tokens=200, page_size=16) for _ in range(2))
    slots = torch.tensor([1, 0], dtype=torch.int32, device=cuda_device)
    for d in (one, many):
        d.prefill(0, prompt(37))
        d.prefill(1, prompt(70, 1))
    tokens = torch.randint(0, 503, (2, 5), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    steps = torch.stack([one.forward(slots, tokens[:, i:i + 1])[:, 0] for i in range(5)], 1)
    assert near(many.forward(slots, tokens), steps)
    assert torch.equal(one.cache.tables, many.cache.tables) and one.cache.lengths.tolist() == [42, 75]


def test_prefill_and_steps_agree(weights, cuda_device):
    """The last prompt token through the cache: only the 4-bit rounding of keys and values differs."""
    a, b = (Kv4Decoder(weights, max_seqs=1, max_tokens=200) for _ in range(2))
    whole = a.prefill(0, prompt(90))
    b.prefill(0, prompt(90)[:-1])
    step = b.forward(torch.zeros(1, dtype=torch.int32, device=cuda_device), prompt(90)[-1:][None].to(cuda_device))
    cosine = torch.nn.functional.cosine_similarity(whole, step[0, 0], dim=0)
    assert float(cosine) > 0.97


def test_branches_share_pages_and_go_their_own_ways(weights, cuda_device):
    d = Kv4Decoder(weights, max_seqs=4, max_tokens=120, page_size=16)
    d.prefill(0, prompt(40))
    used = d.cache.num_pages - d.cache.free_pages()
    d.fork(0, [1, 2, 3])
    assert d.cache.num_pages - d.cache.free_pages() == used == 3
    slots = torch.arange(4, dtype=torch.int32, device=cuda_device)
    same = d.forward(slots, torch.full((4, 1), 7, device=cuda_device))
    assert all(torch.equal(same[0], same[i]) for i in range(1, 4))
    # All four wrote into their copies of the third page; the shared one is free again.
    assert d.cache.num_pages - d.cache.free_pages() == 2 + 4
    alone = Kv4Decoder(weights, max_seqs=1, max_tokens=120, page_size=16)
    alone.prefill(0, prompt(40))
    alone.forward(slots[:1], torch.full((1, 1), 7, device=cuda_device))
    tokens = torch.tensor([[1], [2], [3], [4]], device=cuda_device)
    assert near(d.forward(slots, tokens)[2], alone.forward(slots[:1], tokens[2:3])[0])
    d.release([0, 1])
    d.cache.check()
    assert d.cache.status[1].item() == 2 + 2
    assert near(d.forward(slots[2:3], tokens[:1]), alone.forward(slots[:1], tokens[:1]))


def test_drafts_of_the_model_itself_are_kept(weights):
    target, draft = (Kv4Decoder(weights, max_seqs=3, max_tokens=300, seed=s) for s in (0, 1))
    for d in (target, draft):
        d.prefill(0, prompt(50))
        d.fork(0, [1, 2])
    first, _ = target.sample(target.prefill(0, prompt(50)).expand(3, -1))
    draft.prefill(0, prompt(50))
    tokens, gain = target.generate([0, 1, 2], first, 40, draft=draft, drafts=3)
    assert all(len(t) >= 40 for t in tokens) and all(0 <= x < 503 for t in tokens for x in t)
    assert gain > 3.5  # of 4: the two differ by roundings alone
    # Both caches hold what was kept, but for the last token of each slot.
    held = target.cache.lengths.tolist()
    assert held == draft.cache.lengths.tolist() == [50 + len(t) - 1 for t in tokens]


def test_drafts_of_a_smaller_model(weights):
    small = LlamaWeights(replace(CONFIG, num_hidden_layers=1), weights.embed, weights.layers[:1], weights.norm,
                         weights.lm_head)
    target, draft = Kv4Decoder(weights, max_seqs=2, max_tokens=200), Kv4Decoder(small, max_seqs=2, max_tokens=200)
    logits = torch.stack([target.prefill(s, prompt(20 + s, s)) for s in range(2)])
    for s in range(2):
        draft.prefill(s, prompt(20 + s, s))
    first, _ = target.sample(logits)
    tokens, gain = target.generate([0, 1], first, 20, draft=draft, drafts=2)
    assert 1.0 <= gain <= 3.0
    assert target.cache.lengths.tolist() == [20 + s + len(t) - 1 for s, t in enumerate(tokens)]


def test_retrieval_with_a_full_budget_is_the_dense_attention(weights, cuda_device):
    dense = Kv4Decoder(weights, max_seqs=2, max_tokens=200)
    sparse = Kv4Decoder(weights, max_seqs=2, max_tokens=200, retrieval=RetrievalConfig(budget=500, full_layers=(0,)))
    few = Kv4Decoder(weights, max_seqs=2, max_tokens=200, retrieval=RetrievalConfig(budget=24, full_layers=(0,)))
    for d in (dense, sparse, few):
        d.prefill(0, prompt(80))
        d.fork(0, [1])
    slots = torch.arange(2, dtype=torch.int32, device=cuda_device)
    for i in range(4):
        token = torch.full((2, 1), 11 * i + 1, device=cuda_device)
        want = dense.forward(slots, token)
        assert near(sparse.forward(slots, token), want)
        got = few.forward(slots, token)
        assert torch.isfinite(got).all() and not torch.equal(got, want)
    with pytest.raises(ValueError, match="drafted tokens need dense"):
        sparse.generate([0], torch.zeros(1, dtype=torch.int64), 3, draft=dense)
    tokens, gain = few.generate([0, 1], torch.tensor([1, 2]), 6)
    assert gain == 1.0 and [len(t) for t in tokens] == [6, 6]


def test_a_full_pool_is_reported(weights):
    d = Kv4Decoder(weights, max_seqs=2, max_tokens=64, num_pages=3, page_size=16)
    d.prefill(0, prompt(40))
    with pytest.raises(RuntimeError, match="too few free pages"):
        d.prefill(1, prompt(40))


def test_room_past_max_tokens_is_room(weights, cuda_device):
    """The cache's room is whole pages: tokens of the last page have positions of their own."""
    short, long = Kv4Decoder(weights, max_seqs=1, max_tokens=200), Kv4Decoder(weights, max_seqs=1, max_tokens=256)
    assert short.max_tokens == long.max_tokens == 256
    for d in (short, long):
        d.prefill(0, prompt(199))
    slot = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    tokens = torch.randint(0, 503, (1, 57), generator=torch.Generator().manual_seed(4)).to(cuda_device)
    assert torch.equal(short.forward(slot, tokens[:, :40]), long.forward(slot, tokens[:, :40]))
    assert torch.equal(short.forward(slot, tokens[:, 40:]), long.forward(slot, tokens[:, 40:]))
    assert short.cache.lengths.tolist() == [256]
    whole = Kv4Decoder(weights, max_seqs=1, max_tokens=200)
    assert torch.equal(whole.prefill(0, prompt(256)), long.prefill(0, prompt(256)))
    with pytest.raises(RuntimeError, match="table columns"):
        whole.prefill(0, prompt(257))


def test_room_of_the_sparse_layers_planes(weights, cuda_device):
    d = Kv4Decoder(weights, max_seqs=1, max_tokens=50, page_size=32,
                   retrieval=RetrievalConfig(budget=16, full_layers=(0,)))
    d.prefill(0, prompt(60))
    slot = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for i in range(4):
        assert torch.isfinite(d.forward(slot, torch.full((1, 1), i, device=cuda_device))).all()
    assert d.cache.lengths.tolist() == [64]


def test_sparse_layers_refuse_several_tokens(weights, cuda_device):
    d = Kv4Decoder(weights, max_seqs=2, max_tokens=100, retrieval=RetrievalConfig(budget=16, full_layers=(0,)))
    d.prefill(0, prompt(30))
    slots = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for count in (0, 2, 3):
        with pytest.raises(ValueError, match="one token a step"):
            d.forward(slots, torch.ones((1, count), dtype=torch.int64, device=cuda_device))
    assert d.cache.lengths.tolist() == [30, 0]
    assert all(p.token_count == 30 for p in d.planes.values())
    d.forward(slots, torch.ones((1, 1), dtype=torch.int64, device=cuda_device))
    assert d.cache.lengths.tolist() == [31, 0] and all(p.token_count == 31 for p in d.planes.values())


def test_a_step_without_room_changes_nothing(weights, cuda_device):
    """Branches that find no page for their copies: the prompt they share stays, and the step can be repeated."""
    for retrieval in (None, RetrievalConfig(budget=16, full_layers=(0,))):
        d, other = (Kv4Decoder(weights, max_seqs=3, max_tokens=64, num_pages=n, page_size=16, retrieval=retrieval)
                    for n in (4, 12))
        for x in (d, other):
            x.prefill(0, prompt(40))
            x.fork(0, [1, 2])
        pages, tables = d.cache.pages.clone(), d.cache.tables.clone()
        slots = torch.tensor([1, 2], dtype=torch.int32, device=cuda_device)
        token = torch.full((2, 1), 9, device=cuda_device)
        with pytest.raises(RuntimeError, match="too few free pages"):
            d.forward(slots, token)
        assert torch.equal(d.cache.pages, pages) and torch.equal(d.cache.tables, tables)
        assert all(p.token_count == 40 for p in d.planes.values())
        d.release([2])
        assert near(d.forward(slots[:1], token[:1]), other.forward(slots[:1], token[:1]))
        assert d.cache.lengths.tolist() == [40, 41, 0]


@pytest.mark.parametrize("short_of", ("target", "draft"))
def test_generate_without_room_leaves_both_caches_alike(weights, short_of):
    """The target's and the draft's slots hold the same tokens after a step that one of them had no room for."""
    room = {"target": 5, "draft": 5, short_of: 3}
    target, draft = (Kv4Decoder(weights, max_seqs=1, max_tokens=80, page_size=16, num_pages=room[who], seed=s)
                     for s, who in enumerate(("target", "draft")))
    logits = target.prefill(0, prompt(40))
    draft.prefill(0, prompt(40))
    first, _ = target.sample(logits[None])
    with pytest.raises(RuntimeError, match="too few free pages"):
        target.generate([0], first, 30, draft=draft, drafts=3)
    held = target.cache.lengths.tolist()
    assert held == draft.cache.lengths.tolist() and 40 < held[0] <= 48
    target.cache.check()
    draft.cache.check()


def test_slots_out_of_range_are_refused(weights, cuda_device):
    """An id that is no slot raises, and the other slots of the call keep what they held."""
    for retrieval in (None, RetrievalConfig(budget=16, full_layers=(0,))):
        d = Kv4Decoder(weights, max_seqs=3, max_tokens=100, retrieval=retrieval)
        for s in range(2):
            d.prefill(s, prompt(30 + s))
        pages = d.cache.pages.clone()
        for bad in (7, -3, 1 << 30):
            with pytest.raises((RuntimeError, ValueError), match="out of range or repeated|no prompt"):
                d.forward(torch.tensor([1, bad], dtype=torch.int32, device=cuda_device),
                          torch.zeros((2, 1), dtype=torch.int64, device=cuda_device))
            assert d.cache.lengths.tolist() == [30, 31, 0] and torch.equal(d.cache.pages, pages)
        with pytest.raises((RuntimeError, ValueError), match="out of range or repeated|no prompt"):
            d.generate([0, 9], torch.tensor([1, 2]), 3)
        assert d.cache.lengths.tolist() == [30, 31, 0]


def test_a_prompt_without_room_leaves_no_planes(weights, cuda_device):
    d = Kv4Decoder(weights, max_seqs=1, max_tokens=64, page_size=16,
                   retrieval=RetrievalConfig(budget=16, full_layers=(0,)))
    d.prefill(0, prompt(40))
    with pytest.raises(RuntimeError, match="table columns"):
        d.prefill(0, prompt(65))
    with pytest.raises(ValueError, match="no prompt"):
        d.forward(torch.zeros(1, dtype=torch.int32, device=cuda_device), torch.zeros((1, 1), dtype=torch.int64,
                                                                                     device=cuda_device))
    assert d.cache.lengths.tolist() == [0]


def test_the_default_pool_has_room_for_every_slots_copies(weights, cuda_device):
    """Slots that share their last page, two by two or all four, extend together: a step copies it for each."""
    for pairs, room, held in ((True, 16, 9), (False, 16, 9), (True, 32, 20), (False, 32, 20), (True, 32, 9)):
        d = Kv4Decoder(weights, max_seqs=4, max_tokens=room, page_size=16)
        for s in (0, 2) if pairs else (0,):
            d.prefill(s, prompt(held, s))
        if pairs:
            d.fork(0, [1])
            d.fork(2, [3])
        else:
            d.fork(0, [1, 2, 3])
        slots = torch.arange(4, dtype=torch.int32, device=cuda_device)
        for i in range(room - held):
            d.forward(slots, torch.full((4, 1), i, device=cuda_device))
        assert d.cache.lengths.tolist() == [room] * 4


def test_generate_draws_independent_numbers(weights, monkeypatch):
    """Decoders of the same (default) seed: no random number decides a draft and its verification both."""
    target, draft = (Kv4Decoder(weights, max_seqs=2, max_tokens=200) for _ in range(2))
    for d in (target, draft):
        for s in range(2):
            d.prefill(s, prompt(30))
    drawn = []
    noise, uniform = Kv4Decoder._noise, torch.rand

    def noise_kept(self, *args):
        drawn.append(noise(self, *args))
        return drawn[-1]

    def uniform_kept(*args, **kwargs):
        out = uniform(*args, **kwargs)
        drawn.append(-torch.log1p(-out))
        drawn.append(-torch.log(out))  # either way to exponential numbers
        return out

    monkeypatch.setattr(Kv4Decoder, "_noise", noise_kept)
    monkeypatch.setattr(torch, "rand", uniform_kept)
    first, _ = target.sample(torch.zeros((2, 503), device=target.device))
    target.generate([0, 1], first, 20, draft=draft, drafts=3)
    assert len(drawn) > 20
    for i, a in enumerate(drawn):
        for b in drawn[:i]:
            if a.shape == b.shape and a.shape[1] == 503:
                # Independent fp32 numbers are equal in about one of 10^7 places.
                assert float((a == b).float().mean()) < 0.01


def test_generated_tokens_are_the_targets(cuda_device):
    """First new tokens of many branches through generate, default seeds, a draft model of its own: the target's
    probabilities within five deviations, and a bf16 rounding or two of the logits (2% of a probability)."""
    config = replace(CONFIG, vocab_size=12)
    target = Kv4Decoder(LlamaWeights.random(config, device=cuda_device, std=0.08, seed=5), max_seqs=64, max_tokens=64)
    draft = Kv4Decoder(LlamaWeights.random(replace(config, num_hidden_layers=1), device=cuda_device, std=0.08, seed=6),
                       max_seqs=64, max_tokens=64)
    ids = torch.randint(0, 12, (20,), generator=torch.Generator().manual_seed(0))
    slots = torch.arange(64, dtype=torch.int32, device=cuda_device)
    for d in (target, draft):
        d.prefill(0, ids)
        d.fork(0, list(range(1, 64)))
    lengths = torch.full((64,), 20, device=cuda_device)
    first = torch.full((64,), 3, device=cuda_device)
    logits = target.forward(slots, torch.stack([first, first, first], 1))
    p = logits[0, 0].double().softmax(-1).cpu()
    target.cache.truncate(slots, lengths)
    counts = torch.zeros(12, dtype=torch.float64)
    steps = 120
    for _ in range(steps):
        tokens, _ = target.generate(list(range(64)), first, 2, draft=draft, drafts=2)
        counts += torch.bincount(torch.tensor([t[1] for t in tokens]), minlength=12)
        for d in (target, draft):
            d.cache.truncate(slots, lengths)
    want = p * steps * 64
    assert float(p.max()) < 0.9
    assert ((counts - want).abs() <= 5 * (want * (1 - p)).sqrt() + 0.02 * want + 1).all(), (counts, want)


def test_sampling_arguments_are_checked(weights):
    """Before a token is drawn: a temperature of 0 made every probability NaN, and every token id 0."""
    d = Kv4Decoder(weights, max_seqs=1, max_tokens=64)
    logits = d.prefill(0, prompt(20))[None]
    for temperature in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            d.sample(logits, temperature)
        with pytest.raises(ValueError, match="temperature"):
            d.generate([0], torch.zeros(1, dtype=torch.int64), 3, temperature=temperature)
    with pytest.raises(ValueError, match="drafts must be positive"):
        d.generate([0], torch.zeros(1, dtype=torch.int64), 3, draft=d, drafts=0)
    assert d.cache.lengths.tolist() == [20]


def test_a_draft_of_another_vocabulary_is_refused(weights, cuda_device):
    """Before its ids reach the target's embedding."""
    target = Kv4Decoder(weights, max_seqs=1, max_tokens=64)
    other = Kv4Decoder(LlamaWeights.random(replace(CONFIG, vocab_size=600), device=cuda_device), max_seqs=1,
                       max_tokens=64)
    for d in (target, other):
        d.prefill(0, prompt(20))
    with pytest.raises(ValueError, match="vocabulary"):
        target.generate([0], torch.zeros(1, dtype=torch.int64), 3, draft=other)
    assert target.cache.lengths.tolist() == other.cache.lengths.tolist() == [20]


def test_the_command_runs(cuda_device, capsys):
    main()
    text = capsys.readouterr().out
    assert "two branches kept" in text and "16 more tokens" in text
