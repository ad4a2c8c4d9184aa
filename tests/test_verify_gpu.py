"""Verification of drafted tokens on the GPU: exact against a float32 host model, and its distribution."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from popkv_b200.speculative import verify_drafts, verify_workspace
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


def inputs(n, drafts, vocab, dtype, device, seed, sharp=2.0):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, drafts + 1, vocab, generator=gen) * sharp
    target = logits.softmax(-1).to(dtype)
    draft = (logits[:, :drafts] + 0.5 * torch.randn(n, drafts, vocab, generator=gen)).softmax(-1).to(dtype)
    tokens = (draft.float() / torch.empty(n, drafts, vocab).exponential_(generator=gen)).argmax(-1)
    uniforms = torch.rand(n, drafts, generator=gen)
    noise = torch.empty(n, vocab).exponential_(generator=gen)
    return [t.to(device) for t in (target, tokens.reshape(n, drafts), uniforms, noise, draft)]


def check(target, tokens, uniforms, noise, draft, counts=None):
    got, accepted = verify_drafts(target, tokens, uniforms, noise, draft_probs=draft, counts=counts)
    n, drafts = tokens.shape
    t, u, e = target.float().cpu().numpy(), uniforms.cpu().numpy(), noise.cpu().numpy()
    q = None if draft is None else draft.float().cpu().numpy()
    for i in range(n):
        count = drafts if counts is None else int(counts[i])
        with np.errstate(divide="ignore", over="ignore"):
            want, took = R.verify(t[i], None if q is None else q[i], tokens[i].tolist(), count, u[i], e[i])
        assert got[i].tolist() == want and int(accepted[i]) == took, (i, got[i].tolist(), want)
    return got, accepted


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("n,drafts,vocab", [(1, 1, 1), (1, 4, 7), (3, 2, 1000), (5, 8, 4099), (2, 3, 32000),
                                            (70, 1, 513), (4, 5, 50001)])
@pytest.mark.parametrize("proposal", (True, False))
def test_tokens_match_the_model(cuda_device, dtype, n, drafts, vocab, proposal):
    target, tokens, uniforms, noise, draft = inputs(n, drafts, vocab, dtype, cuda_device, n + drafts + vocab)
    draft = draft if proposal else None
    check(target, tokens, uniforms, noise, draft)
    check(target, tokens, uniforms * 0, noise, draft)  # everything with a probability is accepted
    counts = torch.tensor([i % (drafts + 1) for i in range(n)], dtype=torch.int32, device=cuda_device)
    check(target, tokens, uniforms, noise, draft, counts)


def test_views_and_odd_strides(cuda_device):
    target, tokens, uniforms, noise, draft = inputs(4, 3, 1001, torch.bfloat16, cuda_device, 0)
    wide = torch.zeros(4, 6, 1003, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 1:5, 1:1002] = target
    other = torch.zeros(3, 4, 1007, dtype=torch.bfloat16, device=cuda_device)
    other[:, :, 3:1004] = draft.transpose(0, 1)
    want = verify_drafts(target, tokens, uniforms, noise, draft_probs=draft)
    got = verify_drafts(wide[:, 1:5, 1:1002], tokens, uniforms, noise, draft_probs=other.transpose(0, 1)[:, :, 3:1004])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    strided = verify_drafts(target.transpose(1, 2).contiguous().transpose(1, 2), tokens, uniforms,
                            noise.t().contiguous().t(), draft_probs=draft)
    assert all(torch.equal(a, b) for a, b in zip(strided, want))


def test_ties_zeros_and_ids_out_of_range(cuda_device):
    vocab, dev = 700, cuda_device
    ones = torch.ones(1, vocab, device=dev)
    half = torch.zeros(1, 2, vocab, device=dev)
    half[0, 0, [3, 650]] = 0.5
    half[0, 1, [699, 5]] = 0.5
    no = torch.full((1, 1), 0.75, device=dev)

    def run(target, token, draft, u=no, noise=ones):
        return check(target, torch.tensor([[token]], device=dev), u, noise, draft)[0][0].tolist()

    assert run(half, 7, None) == [3, -1]              # refused: equal ratios go to the lowest id
    assert run(half, 3, None) == [650, -1]            # refused: the draft itself is out
    assert run(half, 3, None, no * 0) == [3, 5]       # accepted: the following row, lowest id
    assert run(half, 3, half[:, :1]) == [3, 5]        # p = q
    assert run(half, -1, None) == [3, -1]             # an id out of range is refused
    assert run(half, vocab, half[:, :1]) == [3, -1]   # and with no residual at all the target's row decides
    assert run(half * 0, 3, None) == [0, -1]          # an empty target: the lowest id
    tiny = half.clone()
    tiny[0, 0, 600] = 1e-30
    assert run(tiny, 9, None, noise=ones * 1e20) == [3, -1]
    spot = ones.clone()
    spot[0, 600] = 1e-38
    assert run(tiny, 9, None, noise=spot) == [600, -1]


def test_no_drafts_samples_the_target(cuda_device):
    target, tokens, uniforms, noise, _ = inputs(9, 0, 999, torch.float32, cuda_device, 5)
    got, accepted = check(target, tokens, uniforms, noise, None)
    assert got.shape == (9, 1) and not accepted.any()
    empty = verify_drafts(target[:0], tokens[:0], uniforms[:0], noise[:0])
    assert empty[0].shape == (0, 1) and empty[1].shape == (0,)


def test_first_token_is_distributed_as_the_target(cuda_device):
    """60000 independent sequences of one draft: the first token's counts within five deviations of p."""
    n, vocab = 60000, 6
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    p = torch.tensor([0.4, 0.05, 0.25, 0.1, 0.0, 0.2], device=cuda_device)
    q = torch.tensor([0.1, 0.3, 0.2, 0.1, 0.2, 0.1], device=cuda_device)
    tokens = torch.multinomial(q, n, replacement=True, generator=gen)[:, None]
    noise = torch.empty(n, vocab, device=cuda_device).exponential_(generator=gen)
    got, accepted = verify_drafts(p.expand(n, 2, vocab), tokens, torch.rand(n, 1, device=cuda_device, generator=gen),
                                  noise, draft_probs=q.expand(n, 1, vocab))
    counts = torch.bincount(got[:, 0], minlength=vocab).double().cpu().numpy()
    want = p.double().cpu().numpy() * n
    assert (np.abs(counts - want) <= 5 * np.sqrt(want * (1 - want / n)) + 1e-9).all(), counts
    rate = float(torch.minimum(p, q).sum())
    assert abs(float(accepted.sum()) - rate * n) <= 5 * (n * rate * (1 - rate)) ** 0.5


def test_calls_on_two_streams(cuda_device):
    sets = [inputs(33, 4, 20001, torch.float32, cuda_device, s) for s in (1, 2)]
    want = [verify_drafts(t, d, u, e, draft_probs=q) for t, d, u, e, q in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                t, d, u, e, q = sets[i]
                got[i].append(verify_drafts(t, d, u, e, draft_probs=q))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_refusals(cuda_device):
    target, tokens, uniforms, noise, draft = inputs(2, 3, 11, torch.float32, cuda_device, 0)
    with pytest.raises(ValueError, match="target_probs must be"):
        verify_drafts(target[:, :3], tokens, uniforms, noise)
    with pytest.raises(ValueError, match="target_probs must be"):
        verify_drafts(target[0], tokens, uniforms, noise)
    with pytest.raises(ValueError, match="uniforms must be"):
        verify_drafts(target, tokens, uniforms[:, :2], noise)
    with pytest.raises(ValueError, match="noise"):
        verify_drafts(target, tokens, uniforms, noise[:, :5])
    with pytest.raises(ValueError, match="draft_probs"):
        verify_drafts(target, tokens, uniforms, noise, draft_probs=draft[:, :2])
    with pytest.raises(ValueError, match="counts"):
        verify_drafts(target, tokens, uniforms, noise, counts=torch.zeros(3, dtype=torch.int32, device=cuda_device))
    with pytest.raises(RuntimeError, match="share an fp32/fp16/bf16"):
        verify_drafts(target, tokens, uniforms, noise, draft_probs=draft.half())
    with pytest.raises(RuntimeError, match="share an fp32/fp16/bf16"):
        verify_drafts(target.double(), tokens, uniforms, noise)
    with pytest.raises(RuntimeError, match="int64"):
        verify_drafts(target, tokens.int(), uniforms, noise)
    with pytest.raises(RuntimeError, match="counts must be int32"):
        verify_drafts(target, tokens, uniforms, noise, counts=torch.zeros(2, dtype=torch.int64, device=cuda_device))
    with pytest.raises(RuntimeError, match="CUDA device"):
        verify_drafts(target, tokens.cpu(), uniforms, noise)


def many_drafts(n, drafts, vocab, device, seed):
    """Inputs whose first refusal falls on a chosen place of each sequence, or on none."""
    target, tokens, uniforms, noise, draft = inputs(n, drafts, vocab, torch.float32, device, seed)
    places = [i * 7919 % (drafts + 1) if i % 3 else drafts - i // 3 % 4 for i in range(n)]
    uniforms = torch.zeros_like(uniforms)
    for i, place in enumerate(places):
        if place < drafts:  # the draft's id of the largest q / p, which is above 1, and the largest u
            tokens[i, place] = (draft[i, place] / target[i, place]).argmax()
            uniforms[i, place] = 1 - 2.0 ** -24
    return places, (target, tokens, uniforms, noise, draft)


@pytest.mark.parametrize("drafts,n,vocab", [(31, 40, 700), (32, 40, 700), (32, 40, 9001), (33, 200, 515), (40, 500, 67), (100, 64, 516),
                                            (1024, 5, 20)])
@pytest.mark.parametrize("proposal", (True, False))
def test_refusals_at_any_place_of_many_drafts(cuda_device, drafts, n, vocab, proposal):
    """More drafts than a warp has lanes: every place may be refused, and every warp writes tokens."""
    places, (target, tokens, uniforms, noise, draft) = many_drafts(n, drafts, vocab, cuda_device, drafts)
    draft = draft if proposal else None
    got, accepted = check(target, tokens, uniforms, noise, draft)
    if proposal:
        assert accepted.tolist() == places
    for _ in range(30):
        again = verify_drafts(target, tokens, uniforms, noise, draft_probs=draft)
        assert torch.equal(again[0], got) and torch.equal(again[1], accepted)


@pytest.mark.parametrize("given", (True, False))
def test_verification_in_a_graph(cuda_device, given):
    """Captured with a workspace of its own or the call's, and replayed on new inputs; one workspace for several sizes."""
    sets = [inputs(6, 4, 5003, torch.float32, cuda_device, s) for s in range(4)]
    held = [t.clone() for t in sets[0]]
    workspace = verify_workspace(9, cuda_device) if given else None

    def call(t, d, u, e, q):
        return verify_drafts(t, d, u, e, draft_probs=q, workspace=workspace)

    call(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*held)
    for s in sets:
        for to, new in zip(held, s):
            to.copy_(new)
        graph.replay()
        want = verify_drafts(*s[:4], draft_probs=s[4])
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        few = [t[:2] for t in s]
        got = call(*few)
        assert torch.equal(got[0], want[0][:2]) and torch.equal(got[1], want[1][:2])
    if given:
        assert not workspace.any()
        with pytest.raises(ValueError, match="workspace"):
            verify_drafts(*held[:4], draft_probs=held[4], workspace=workspace[:12])
    del graph
