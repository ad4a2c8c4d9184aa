"""The 4-bit paged KV cache on the GPU against a host model.

Bytes and tables are compared exactly.  Attention is compared with a 64-bit softmax over the
values that the cached bytes stand for.  Its bound: the output's own rounding (half an ulp of
fp16 or bf16, 2^-11 or 2^-8 of the value at most), plus the rounding of each token's weight
p * delta to fp16, at most 2^-11 of a value's distance from its group's low, that is at most
2^-11 * 2 max|v|; plus the fp32 logits: their error is at most about (128 + 32) * 2^-24 *
sum|q k| * scale, below 1e-5 for these inputs (sum|q k| * scale <= 1024 here), and shifts an
output by at most twice that times max|v|; exp is good to 2^-21.  1e-4 * max|v| covers the
last three.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from popkv_b200.kv4 import Kv4Cache
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu

ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(device, lengths, *, kv_heads=2, page=16, group=32, layers=1, max_tokens=None, spare=3, max_seqs=None,
         layer=0, seed=0):
    """A cache whose sequences hold random tokens, on pages in mixed order."""
    gen = torch.Generator().manual_seed(seed + sum(lengths) + page)
    n = len(lengths)
    max_tokens = max_tokens or max(lengths) + 64
    pages = sum(-(-t // page) for t in lengths) + spare
    cache = Kv4Cache(pages, kv_heads=kv_heads, layers=layers, max_seqs=max_seqs or n, max_tokens=max_tokens,
                     page_size=page, dim_group_size=group, device=device)
    # Hand out the pages a few tokens at a time, so that sequences interleave.
    left = list(lengths)
    while any(left):
        step = [min(t, page + 5) for t in left]
        cache.extend(list(range(n)), torch.tensor(step, dtype=torch.int32, device=device))
        most = max(step)
        x = torch.randn(2, n, most, kv_heads, 128, generator=gen) * torch.exp(torch.randn(128, generator=gen) * 0.5)
        cache.write(x[0].to(device), x[1].to(device), seqs=list(range(n)), layer=layer,
                    counts=torch.tensor(step, dtype=torch.int32, device=device))
        left = [t - s for t, s in zip(left, step)]
    cache.check()
    return cache


def expect(cache, host, queries, positions_of, *, layer=0, scale=128 ** -0.5):
    """float64 outputs [rows..., q_heads, 128] and max|v|; positions_of(index) lists a row's tokens, head by head."""
    q = queries.double().cpu().numpy()
    out = np.zeros(q.shape)
    q_heads = q.shape[-2]
    most = 0.0
    memo = {}
    for at in np.ndindex(*q.shape[:-1]):
        seq, positions = positions_of(at)
        head = at[-1] // (q_heads // cache.kv_heads)
        rows = []
        for t in positions:
            key = (seq, head, int(t))
            if key not in memo:
                memo[key] = host.get(layer, seq, head, int(t))
            rows.append(memo[key])
        if rows:
            keys, values = np.stack([k for k, _ in rows]), np.stack([v for _, v in rows])
            most = max(most, np.abs(values).max())
            out[at] = R.attention(q[at], keys, values, scale)
    return out, most


def close(got, want, most):
    bound = ULP[got.dtype] * np.abs(want) + (2.0 ** -10 + 1e-4) * most
    error = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(error).all()
    assert (error <= bound).all(), f"error {error.max():.3g}, {(error / np.maximum(bound, 1e-30)).max():.3g} of the bound"


def random_queries(shape, dtype, device, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


# -- rows ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("page,prior,tokens,heads", [(16, 0, 1, 1), (16, 5, 30, 3), (64, 63, 2, 2), (256, 250, 21, 5)])
def test_write_and_read_match_the_model(cuda_device, dtype, group, page, prior, tokens, heads):
    cache = make(cuda_device, [prior + tokens] * 2, kv_heads=heads, page=page, group=group, layers=2, layer=1)
    host = R.HostCache.like(cache)
    gen = torch.Generator().manual_seed(tokens + group)
    qkv = torch.randn(2, tokens, 3 * heads + 1, 128, generator=gen).to(dtype).to(cuda_device)
    keys, values = qkv[:, :, 1:1 + heads], qkv[:, :, 1 + 2 * heads:]
    cache.write(keys, values, seqs=[1, 0], layer=1)
    k, v = keys.float().cpu().numpy(), values.float().cpu().numpy()
    for i, seq in enumerate((1, 0)):
        for t in range(tokens):
            for h in range(heads):
                host.put(1, seq, h, prior + t, k[i, t, h], v[i, t, h])
    host.same(cache)
    # A reading that starts before the rows and ends past the sequence.
    start = max(0, prior - 3)
    for out in (torch.float32, dtype):
        got = cache.read([0, 1, -1], start=start, tokens=tokens + 9, layer=1, dtype=out)
        for which in range(2):
            want = np.zeros((3, tokens + 9, heads, 128))
            for s in range(2):
                for t in range(start, prior + tokens):
                    for h in range(heads):
                        want[s, t - start, h] = host.get(1, s, h, t)[which]
            assert torch.equal(got[which].cpu(), torch.from_numpy(want).float().to(out))


def test_write_odd_values(cuda_device):
    """NaN, infinities, constants, tiny ranges and fp16's denormals are stored as the formula says."""
    cache = make(cuda_device, [9], kv_heads=1)
    host = R.HostCache.like(cache)
    x = torch.zeros(1, 9, 1, 128)
    x[0, 0] = float("nan")
    x[0, 1, 0, ::2] = float("inf")
    x[0, 2, 0, 1::3] = -float("inf")
    x[0, 3] = 7.3
    x[0, 4, 0, 5] = 1e-7
    x[0, 5] = torch.linspace(-1e30, 1e30, 128)
    x[0, 6] = torch.linspace(-2e-7, 3e-7, 128)
    x[0, 7, 0, :40] = float("nan")
    x[0, 8] = torch.linspace(-65504, 65504, 128)
    cache.write(x.to(cuda_device), x.flip(-1).to(cuda_device), seqs=[0])
    for t in range(9):
        host.put(0, 0, 0, t, x[0, t, 0].numpy(), x[0, t, 0].flip(0).numpy())
    host.same(cache)
    keys, values = cache.read([0], tokens=9, dtype=torch.float32)
    assert torch.isfinite(keys).all() and torch.isfinite(values).all()


def test_write_rounds_the_range_as_documented(cuda_device):
    """Ranges whose product with 1/15 and quotient by 15 round to different fp16 deltas."""
    r = np.random.default_rng(0).uniform(1.0, 30.0, 1 << 21).astype(np.float32)
    r = r[(r * (np.float32(1) / np.float32(15))).astype(np.float16) != (r / np.float32(15)).astype(np.float16)][:64]
    assert len(r) >= 32
    x = torch.rand(1, len(r), 1, 128, generator=torch.Generator().manual_seed(1)) * torch.from_numpy(r)[:, None, None]
    x[..., 0] = 0.0
    x[..., 127] = torch.from_numpy(r)[:, None]
    cache = Kv4Cache(8, kv_heads=1, max_seqs=1, max_tokens=128, dim_group_size=128, page_size=16, device=cuda_device)
    cache.extend([0], len(r))
    cache.write(x.to(cuda_device), -x.to(cuda_device), seqs=[0])
    keys, values = cache.read([0], tokens=len(r), dtype=torch.float32)
    for got, given in ((keys, x), (values, -x)):
        n, low, delta = R.quantise(given.numpy(), 128)
        want = low.astype(np.float32) + n.astype(np.float32) * delta.astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want)


def test_write_counts_padding_and_unaligned_views(cuda_device):
    cache = make(cuda_device, [20, 33, 7])
    host = R.HostCache.like(cache)
    flat = torch.randn(3 * 4 * 2 * 131 + 1, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    keys = flat[1:].view(3, 4, 2, 131)[..., 1:129]  # rows that start on odd elements
    values = keys.transpose(0, 1).contiguous().transpose(0, 1)
    cache.write(keys, values, seqs=[2, -1, 1], counts=torch.tensor([3, 4, 0], dtype=torch.int32, device=cuda_device))
    for t in range(3):
        for h in range(2):
            host.put(0, 2, h, 4 + t, keys[0, t, h].float().cpu().numpy(), values[0, t, h].float().cpu().numpy())
    host.same(cache)
    cache.write(keys[:, 0], values[:, 0], seqs=[99, 0, -5])  # ids out of range: nothing is written
    for h in range(2):
        host.put(0, 0, h, 19, keys[1, 0, h].float().cpu().numpy(), values[1, 0, h].float().cpu().numpy())
    host.same(cache)


# -- attention ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype,group,page,heads,per,q_len,lengths", [
    (torch.bfloat16, 32, 16, 1, 1, 1, [1]),
    (torch.float16, 32, 64, 2, 4, 1, [0, 1, 15, 16, 17, 130]),
    (torch.float16, 64, 32, 3, 3, 2, [2, 31, 33, 1]),
    (torch.float16, 128, 128, 1, 7, 3, [127, 129, 5]),
    (torch.bfloat16, 64, 256, 2, 8, 1, [300, 255]),
    (torch.float16, 32, 64, 1, 4, 5, [200, 64, 3]),
    (torch.float16, 64, 16, 2, 1, 9, [77]),
    (torch.float16, 32, 16, 1, 12, 7, [140, 12]),
    (torch.bfloat16, 128, 16, 1, 2, 40, [61]),
])
def test_attention_matches_64_bits(cuda_device, dtype, group, page, heads, per, q_len, lengths):
    cache = make(cuda_device, lengths, kv_heads=heads, page=page, group=group)
    host = R.HostCache.like(cache)
    queries = random_queries((len(lengths), q_len, heads * per, 128), dtype, cuda_device, len(lengths))
    got = cache.attention(queries, seqs=list(range(len(lengths))))
    want, most = expect(cache, host, queries, lambda at: (at[0], range(max(0, lengths[at[0]] - q_len + at[1] + 1))))
    close(got, want, most)
    assert torch.equal(got, cache.attention(queries, seqs=list(range(len(lengths)))))
    for i, t in enumerate(lengths):  # rows that see no token
        for j in range(q_len):
            if t - q_len + j + 1 <= 0:
                assert not got[i, j].any()


def test_attention_long_and_split(cuda_device):
    """Long rows, which several CTAs share, with peaked and flat softmaxes."""
    lengths = [5003, 1, 2048]
    cache = make(cuda_device, lengths, kv_heads=1, page=64)
    host = R.HostCache.like(cache)
    queries = random_queries((3, 1, 4, 128), torch.float16, cuda_device, 3)
    queries[0, 0, 1] *= 0.0
    queries[0, 0, 2] *= 6.0
    got = cache.attention(queries, seqs=[0, 1, 2])
    want, most = expect(cache, host, queries, lambda at: (at[0], range(lengths[at[0]])))
    close(got, want, most)


@pytest.mark.parametrize("dtype,group,page,heads,per,q_len", [
    (torch.float16, 32, 16, 2, 4, 1),
    (torch.bfloat16, 64, 64, 2, 3, 1),
    (torch.float16, 128, 16, 4, 1, 1),
    (torch.float16, 32, 32, 2, 7, 1),
    (torch.float16, 128, 64, 2, 4, 4),
    (torch.float16, 64, 16, 2, 2, 5),
    (torch.bfloat16, 32, 64, 2, 4, 5),
    (torch.float16, 64, 32, 2, 5, 4),
    (torch.float16, 32, 16, 1, 8, 5),
])
def test_attention_of_many_uneven_sequences(cuda_device, dtype, group, page, heads, per, q_len):
    """More (sequence, head) pairs than CTAs of an SM take in a wave, some of them cut into parts."""
    lengths = [(53 * i) % 140 if i % 23 else 900 * (i % 4) + 33 for i in range(150)]
    cache = make(cuda_device, lengths, kv_heads=heads, page=page, group=group)
    host = R.HostCache.like(cache)
    queries = random_queries((150, q_len, heads * per, 128), dtype, cuda_device, group + q_len)
    got = cache.attention(queries, seqs=list(range(150)))
    some = [0, 1, 23, 46, 69, 70, 92, 115, 138, 149]
    want, most = expect(cache, host, queries[some],
                        lambda at: (some[at[0]], range(max(0, lengths[some[at[0]]] - q_len + at[1] + 1))))
    close(got[some], want, most)
    # A sequence's result is the same to rounding in a batch of its own, where the work is cut in another way.
    alone = [cache.attention(queries[i:i + 1], seqs=[i]) for i in range(150)]
    close(got, torch.cat(alone).double().cpu().numpy(), 2 * most)
    assert torch.equal(got, cache.attention(queries, seqs=list(range(150))))


def test_attention_counts_padding_and_strides(cuda_device):
    lengths = [40, 18, 2]
    cache = make(cuda_device, lengths, kv_heads=2, page=16)
    host = R.HostCache.like(cache)
    fused = random_queries((4, 3, 12, 128), torch.float16, cuda_device, 5)
    queries = fused[:, :, 2:10]
    seqs, counts = [2, -1, 0, 1], [3, 3, 1, 0]
    out = cache.attention(queries, seqs=seqs, counts=torch.tensor(counts, dtype=torch.int32, device=cuda_device))

    def positions(at):
        s, c = seqs[at[0]], counts[at[0]]
        return s, range(max(0, lengths[s] - c + at[1] + 1)) if s >= 0 and at[1] < c else range(0)

    want, most = expect(cache, host, queries, positions)
    close(out, want, most)
    assert not out[1].any() and not out[3].any() and not out[2, 1:].any() and not out[0, 0].any()
    one = cache.attention(queries[:, 0], seqs=seqs, softmax_scale=0.25)
    want, most = expect(cache, host, queries[:, 0],
                        lambda at: (seqs[at[0]], range(lengths[seqs[at[0]]] if seqs[at[0]] >= 0 else 0)), scale=0.25)
    close(one, want, most)


@pytest.mark.parametrize("stale", (0x7FFF, 0x7C00, -0x400, 0x7BFF))  # NaN, inf, -inf, the largest value
def test_attention_ignores_what_lies_past_the_end(cuda_device, stale):
    """Stale bytes behind a sequence's end and page ids out of range."""
    cache = make(cuda_device, [21, 50], kv_heads=2, page=16)
    host = R.HostCache.like(cache)
    before = cache.attention(random_queries((2, 2, 4, 128), torch.float16, cuda_device, 8), seqs=[0, 1])
    for seq, length in ((0, 21), (1, 50)):
        page = int(cache.table[seq, (length - 1) // 16])
        tile = cache.pages[0, page].view(2, -1)
        for r in range(length % 16, 16):
            tile[:, r * 64:(r + 1) * 64] = 255
            tile[:, 1024 + r * 64:1024 + (r + 1) * 64] = 255
            tile.view(torch.int16)[:, 1024 + r * 16:1024 + (r + 1) * 16] = stale
    queries = random_queries((2, 2, 4, 128), torch.float16, cuda_device, 8)
    assert torch.equal(before, cache.attention(queries, seqs=[0, 1]))
    picked = torch.tensor([3, 20, 21, 22, 49, 50, 63], device=cuda_device).expand(2, 4, 7)
    got = cache.attention_selected(queries[:, 0], picked, seqs=[0, 1])
    want, most = expect(cache, host, queries[:, 0], lambda at: (at[0], [t for t in (3, 20, 21, 22, 49)
                                                                        if t < (21, 50)[at[0]]]))
    close(got, want, most)
    # Tokens of a missing page do not exist.
    cache.table[1, 1] = -1
    got = cache.attention(queries, seqs=[0, 1])

    def positions(at):
        last = (21, 50)[at[0]] - 2 + at[1] + 1
        return at[0], [t for t in range(last) if at[0] == 0 or not 16 <= t < 32]

    want, most = expect(cache, host, queries, positions)
    close(got, want, most)
    cache.table[1, 2] = cache.num_pages + 7
    got = cache.attention(queries, seqs=[0, 1])
    want, most = expect(cache, host, queries,
                        lambda at: (at[0], [t for t in positions(at)[1] if at[0] == 0 or t < 32 or t >= 48]))
    close(got, want, most)


def chunk_coded(device, lengths, *, kv_heads, page, group):
    """A cache whose value of a token is 1 in the dim (number of its 32 tokens + head) % 128 and 0 elsewhere, so
    that an output is the weight of each 32 tokens and lost ones leave a hole of their own."""
    cache = Kv4Cache(sum(-(-t // page) for t in lengths), kv_heads=kv_heads, max_seqs=len(lengths),
                     max_tokens=max(lengths), page_size=page, dim_group_size=group, device=device)
    gen = torch.Generator().manual_seed(len(lengths))
    for s, tokens in enumerate(lengths):
        if not tokens:
            continue
        cache.extend([s], tokens)
        dims = (torch.arange(tokens)[:, None] // 32 + torch.arange(kv_heads)) % 128
        values = torch.nn.functional.one_hot(dims, 128).half()
        keys = torch.randn(tokens, kv_heads, 128, generator=gen).half()
        cache.write(keys[None].to(device), values[None].to(device), seqs=[s])
    cache.check()
    return cache


def chunk_weights(query, positions, group, scale=128 ** -0.5):
    """float64 outputs of a query [128] over tokens of its KV head, and the bound on a kernel's difference.

    Numbers enter the outputs as n - 8, with weights p * delta rounded to fp16: 2^-11 of |n - 8| * delta <=
    8/15 for the tokens whose 1 lies in a dim's group (elsewhere delta is 0 and the value exact).  The output
    rounds by 2^-11 of itself, or half an fp16 denormal.  2^-15 covers the logits (below 1e-6, see above), exp2 and the
    products' truncated additions (2^-23 of a partial sum below 0.6 for each of up to 2000).
    """
    keys, values, head = query[1]
    k, v = keys[:, head][positions], values[:, head][positions]
    p = torch.softmax(k @ query[0] * scale, 0)
    mass = (p @ v).view(-1, group).sum(-1).repeat_interleave(group)
    want = p @ v
    return want, 2.0 ** -11 * (8 / 15) * mass + 2.0 ** -11 * want + 2.0 ** -15


@pytest.mark.parametrize("lengths,heads,per,q_len,page,group", [
    ([20011], 1, 4, 1, 64, 32), ([9001], 1, 8, 1, 16, 64), ([6003], 1, 4, 4, 64, 128), ([6003], 1, 4, 5, 64, 32),
    ([4099], 1, 4, 10, 32, 32), ([777, 5003, 64, 0, 3001] * 7, 2, 4, 1, 16, 32),
    ([777, 3001, 64, 0, 2005] * 13, 2, 3, 2, 64, 64), ([777, 2001, 64, 0, 1005] * 13, 2, 4, 5, 64, 32)])
def test_attention_leaves_no_chunk_out(cuda_device, lengths, heads, per, q_len, page, group):
    """A bound that 32 tokens left out exceed by far wherever a segment is cut."""
    cache = chunk_coded(cuda_device, lengths, kv_heads=heads, page=page, group=group)
    n = len(lengths)
    queries = 0.3 * torch.randn(n, q_len, heads * per, 128, generator=torch.Generator().manual_seed(7))
    queries = queries.half().to(cuda_device)
    got = cache.attention(queries, seqs=list(range(n))).double()
    index = torch.stack([torch.randperm(max(lengths), generator=torch.Generator().manual_seed(h))
                         for h in range(heads * per)]).to(cuda_device)
    picked = cache.attention_selected(queries[:, 0], index.expand(n, -1, -1), seqs=list(range(n))).double()
    for s in range(n):
        if not lengths[s]:
            assert not got[s].any() and not picked[s].any()
            continue
        keys, values = (x[0].double() for x in cache.read([s], tokens=lengths[s], dtype=torch.float32))
        for h in range(heads * per):
            for j in range(q_len):
                seen = slice(0, max(0, lengths[s] - q_len + j + 1))
                query = queries[s, j, h].double(), (keys, values, h // per)
                want, bound = chunk_weights(query, seen, group)
                error = (got[s, j, h] - want).abs()
                assert (error <= bound).all(), (s, j, h, float((error / bound).max()))
            query = queries[s, 0, h].double(), (keys, values, h // per)
            want, bound = chunk_weights(query, slice(0, lengths[s]), group)
            error = (picked[s, h] - want).abs()
            assert (error <= bound).all(), (s, h, float((error / bound).max()))
            # What the bound is for: the largest and the smallest hole that 32 tokens would leave.
            k = keys[:, h // per]
            p = torch.softmax(k @ queries[s, 0, h].double() * 128 ** -0.5, 0)
            holes = torch.stack([c.sum() for c in p.split(32) if len(c) == 32]) if lengths[s] >= 32 else p[:0]
            assert not len(holes) or float(holes.min()) > 4 * float(bound.max())


def test_attention_of_extreme_logits(cuda_device):
    """Large logits, equal logits, tiny and large values; a NaN query spoils its own row alone."""
    cache = make(cuda_device, [70], kv_heads=1, page=64)
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(1, 70, 1, 128, generator=gen)
    cache.write((x * 30).to(cuda_device), (x.flip(1) * 900).to(cuda_device), seqs=[0])
    host = R.HostCache.like(cache)
    queries = random_queries((1, 1, 8, 128), torch.bfloat16, cuda_device, 1)
    queries[0, 0, 1] *= 100
    queries[0, 0, 2] *= 1e-30
    queries[0, 0, 3] = 0
    queries[0, 0, 4, 1:] = 0  # one dim alone
    queries[0, 0, 5, 7] = 1e-20  # a dim far below the others
    got = cache.attention(queries, seqs=[0], softmax_scale=0.01)
    want, most = expect(cache, host, queries, lambda at: (0, range(70)), scale=0.01)
    # Row 1: sum|q k| * scale reaches 2500; about 16 roundings of 2^-24 of it, twice: 5e-3 * max|v|.
    bound = ULP[got.dtype] * np.abs(want) + (2.0 ** -10 + 1e-4) * most
    bound[0, 0, 1] += 5e-3 * most
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    spoiled = queries.clone()
    spoiled[0, 0, 6, 3] = float("nan")
    other = cache.attention(spoiled, seqs=[0], softmax_scale=0.01)
    assert torch.isnan(other[0, 0, 6]).all()
    keep = [h for h in range(8) if h != 6]
    assert torch.equal(other[0, 0, keep], got[0, 0, keep])


def test_attention_of_small_deltas_beside_large(cuda_device):
    """Values whose groups' steps differ by five orders of magnitude: p * delta must not be lost."""
    cache = make(cuda_device, [64], kv_heads=1, page=64)
    gen = torch.Generator().manual_seed(6)
    values = torch.randn(1, 64, 1, 128, generator=gen) * 1e-3
    values[0, 10] *= 1e5
    keys = torch.randn(1, 64, 1, 128, generator=gen)
    queries = random_queries((1, 1, 4, 128), torch.float16, cuda_device, 2)
    keys[0, 10, 0] = -8 * queries[0, 0].float().cpu().mean(0)  # the large one is hardly seen
    cache.write(keys.to(cuda_device), values.to(cuda_device), seqs=[0])
    host = R.HostCache.like(cache)
    got = cache.attention(queries, seqs=[0])
    want, _ = expect(cache, host, queries, lambda at: (0, range(64)))
    # p of the large token weighs its values: the bound's max|v| is over p * |v|, at most the largest
    # small value plus what the large token adds to an output.
    most = np.abs(want).max() + 5e-3
    close(got, want, most)


@pytest.mark.parametrize("dtype,group,page,heads,per,selected", [
    (torch.bfloat16, 32, 16, 1, 1, 1), (torch.float16, 32, 64, 2, 4, 37), (torch.float16, 64, 32, 2, 3, 130),
    (torch.float16, 128, 128, 1, 8, 300),
])
@pytest.mark.parametrize("masked", (False, True))
def test_selected_matches_64_bits(cuda_device, dtype, group, page, heads, per, selected, masked):
    lengths = [333, 12, 0]
    cache = make(cuda_device, lengths, kv_heads=heads, page=page, group=group)
    host = R.HostCache.like(cache)
    gen = torch.Generator().manual_seed(selected)
    queries = random_queries((3, heads * per, 128), dtype, cuda_device, selected)
    # Any order, repeats, and positions that are negative or past the end.
    indices = torch.randint(-3, 340, (3, heads * per, selected), generator=gen)
    valid = torch.rand(indices.shape, generator=gen) < 0.7
    valid[0, 0] = False
    got = cache.attention_selected(queries, indices.to(cuda_device), seqs=[0, 1, 2],
                                   valid_mask=valid.to(cuda_device) if masked else None)

    def positions(at):
        picked = indices[at][valid[at]] if masked else indices[at]
        return at[0], [int(t) for t in picked if 0 <= t < lengths[at[0]]]

    want, most = expect(cache, host, queries, positions)
    close(got, want, most)
    assert not got[2].any()


def test_selected_all_tokens_is_the_attention(cuda_device):
    cache = make(cuda_device, [700], kv_heads=2, page=64)
    queries = random_queries((1, 8, 128), torch.float16, cuda_device, 9)
    indices = torch.stack([torch.randperm(700, generator=torch.Generator().manual_seed(h)) for h in range(8)])[None]
    got = cache.attention_selected(queries, indices.to(cuda_device), seqs=[0])
    host = R.HostCache.like(cache)
    want, most = expect(cache, host, queries, lambda at: (0, range(700)))
    close(got, want, most)
    close(cache.attention(queries, seqs=[0]), want, most)
    nothing = cache.attention_selected(queries, indices[..., :0].to(cuda_device), seqs=[0])
    assert not nothing.any()


def test_attention_beyond_32_bit_offsets(cuda_device):
    """A pool of 5 GB, its last pages and layer in use."""
    cache = Kv4Cache(61000, kv_heads=4, layers=2, max_seqs=2, max_tokens=200, page_size=64, dim_group_size=32,
                     device=cuda_device)
    cache.refs[:60990] = 1  # somebody else's
    cache.extend([1], 150)
    x = torch.randn(2, 1, 150, 4, 128, generator=torch.Generator().manual_seed(2)).half().to(cuda_device)
    cache.write(x[0], x[1], seqs=[1], layer=1)
    cache.check()
    assert int(cache.table[1, 0]) == 60990
    keys, values = cache.read([1], tokens=150, layer=1, dtype=torch.float32)
    k64, v64 = keys[0].double().cpu().numpy(), values[0].double().cpu().numpy()
    for h in range(4):
        n, low, delta = R.quantise(x[0, 0, :, h].float().cpu().numpy(), 32)
        np.testing.assert_array_equal(k64[:, h], R.values_of(n, low, delta, 32).astype(np.float32))
    queries = random_queries((1, 16, 128), torch.float16, cuda_device, 3)
    got = cache.attention(queries, seqs=[1], layer=1)
    q = queries.double().cpu().numpy()
    want = np.stack([R.attention(q[0, h], k64[:, h // 4], v64[:, h // 4], 128 ** -0.5) for h in range(16)])[None]
    close(got, want, np.abs(v64).max())
    picked = torch.arange(150, device=cuda_device).expand(1, 16, 150)
    close(cache.attention_selected(queries, picked, seqs=[1], layer=1), want, np.abs(v64).max())
    # A copy on write into the pool's end.
    cache.fork([1], [0])
    cache.extend([0], 1)
    cache.check()
    assert int(cache.table[0, 2]) == 60993 and torch.equal(cache.pages[1, 60993], cache.pages[1, 60992])


def test_attention_many_sequences_and_streams(cuda_device):
    """More (sequence, head) pairs than CTAs, on a side stream, while another stream does the same."""
    lengths = [(37 * i) % 200 for i in range(300)]
    cache = make(cuda_device, lengths, kv_heads=2, page=16)
    queries = random_queries((300, 4, 128), torch.bfloat16, cuda_device, 0)
    want = cache.attention(queries, seqs=list(range(300)))
    seqs = torch.arange(300, dtype=torch.int32, device=cuda_device)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(cache.attention(queries, seqs=seqs))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    host = R.HostCache.like(cache)
    some = [0, 1, 2, 150, 299]
    got, most = expect(cache, host, queries[some], lambda at: (some[at[0]], range(lengths[some[at[0]]])))
    close(want[some], got, most)


def test_decode_step_in_a_graph(cuda_device):
    """extend, write and attention captured once and replayed: lengths are read on the device."""
    cache = make(cuda_device, [14, 30], kv_heads=2, page=16, spare=8)
    twin = make(cuda_device, [14, 30], kv_heads=2, page=16, spare=8)
    assert torch.equal(cache.pages, twin.pages)
    seqs = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
    x = torch.randn(3, 2, 8, 128, generator=torch.Generator().manual_seed(3)).half().to(cuda_device)
    q, k, v = x[0].clone(), x[1, :, :2].clone(), x[2, :, :2].clone()

    def step(c):
        c.extend(seqs, 1)
        c.write(k, v, seqs=seqs)
        return c.attention(q, seqs=seqs)

    snapshot = cache.tables.clone(), cache.pages.clone()
    step(cache)
    cache.tables.copy_(snapshot[0])
    cache.pages.copy_(snapshot[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(5):
        k.copy_(x[1, :, :2] * (i + 1))
        graph.replay()
        assert torch.equal(out, step(twin))
    cache.check()
    assert torch.equal(cache.tables, twin.tables) and torch.equal(cache.pages, twin.pages)


# -- pages --------------------------------------------------------------------------
def filled(device, num_pages, *, max_seqs=6, page=16, layers=2, max_tokens=160):
    cache = Kv4Cache(num_pages, kv_heads=2, layers=layers, max_seqs=max_seqs, max_tokens=max_tokens, page_size=page,
                     device=device)
    cache.pages.random_(0, 256)
    return cache


@pytest.mark.parametrize("page,num_pages,seed", [(16, 40, 0), (16, 64, 1), (32, 30, 2), (64, 2100, 3), (16, 5000, 4)])
def test_page_operations_follow_the_model(cuda_device, page, num_pages, seed):
    """Random sequences of extend, fork, truncate, free and compact."""
    rng = np.random.default_rng(seed)
    layers = 2 if num_pages < 1000 else 1
    cache = filled(cuda_device, num_pages, page=page, layers=layers, max_tokens=10 * page)
    host = R.HostCache.like(cache)
    for step in range(60):
        op = rng.integers(5)
        k = int(rng.integers(1, 7))
        some = rng.permutation(6)[:k].tolist()
        if op == 0 or step < 4:
            counts = rng.integers(0, 3 * page, k).tolist()
            fine = host.extend(some, counts)
            cache.extend(some, torch.tensor(counts, dtype=torch.int32, device=cuda_device))
            if fine:
                cache.check()
            else:
                with pytest.raises(RuntimeError, match="too few free pages"):
                    cache.check()
        elif op == 1:
            parents = rng.integers(0, 6, k).tolist()
            host.fork(parents, some)
            cache.fork(parents, some)
        elif op == 2:
            lengths = rng.integers(-3, 10 * page, k).tolist()
            host.truncate(some, lengths)
            cache.truncate(some, torch.tensor(lengths, device=cuda_device))
        elif op == 3:
            host.truncate(some[:1], [0])
            cache.free(some[:1])
        else:
            live, moved = host.compact()
            cache.compact()
            assert cache.status[1:3].tolist() == [live, moved]
        if num_pages < 1000 or step % 10 == 9:
            host.same(cache)
        else:
            host.same_tables(cache)
        assert cache.free_pages() == int((host.refs == 0).sum())
    cache.check()


def test_extend_many_pages_at_once(cuda_device):
    cache = filled(cuda_device, 9000, max_seqs=300, layers=1, max_tokens=2000 * 16)
    host = R.HostCache.like(cache)
    rng = np.random.default_rng(7)
    cache.refs[torch.from_numpy(rng.permutation(9000)[:1500]).to(cuda_device)] = 1
    host.refs = cache.refs.cpu().numpy().copy()
    seqs = rng.permutation(300).tolist()
    counts = [31999 if i == 5 else int(rng.integers(0, 200)) for i in range(300)]
    assert host.extend(seqs, counts)
    cache.extend(seqs, torch.tensor(counts, dtype=torch.int32, device=cuda_device))
    cache.check()
    host.same_tables(cache)
    others = [s for i, s in enumerate(seqs) if i != 5]
    assert host.extend(others, [16] * 299)
    cache.extend(others, 16)
    cache.check()
    host.same_tables(cache)
    assert not host.extend([seqs[5]], [17])
    cache.extend([seqs[5]], 17)
    with pytest.raises(RuntimeError, match="table columns"):
        cache.check()
    host.same_tables(cache)


def test_a_failed_extend_changes_nothing(cuda_device):
    cache = filled(cuda_device, 10)
    cache.extend([0, 1], 40)
    cache.fork([0], [2])
    host = R.HostCache.like(cache)
    cache.extend([2, 3], torch.tensor([1, 100], dtype=torch.int32, device=cuda_device))  # 1 + 7 pages of 4
    with pytest.raises(RuntimeError, match="too few free pages"):
        cache.check()
    host.same(cache)
    cache.extend([3], 1 << 30)
    with pytest.raises(RuntimeError, match="table columns"):
        cache.check()
    host.same(cache)
    cache.check()


def test_pages_shared_by_all_extenders(cuda_device):
    """Two holders of a partly filled page that extend together: both get copies, the page is free again."""
    cache = filled(cuda_device, 12)
    cache.extend([0], 20)
    cache.fork([0], [1])
    host = R.HostCache.like(cache)
    last = int(cache.table[0, 1])
    assert host.extend([0, 1], [1, 1])
    cache.extend([0, 1], 1)
    cache.check()
    host.same(cache)
    assert int(cache.refs[last]) == 0


def test_repeated_and_out_of_range_ids(cuda_device):
    cache = filled(cuda_device, 30)
    host = R.HostCache.like(cache)
    cache.extend([0, 0, 9, -1], 20)
    with pytest.raises(RuntimeError, match="out of range or repeated"):
        cache.check()
    host.extend([0], [20])
    host.same_tables(cache)
    cache.extend([1, -1], 5)
    cache.check()
    host.extend([1], [5])
    cache.fork([0, 7, 0], [2, 3, 2])
    with pytest.raises(RuntimeError, match="out of range or repeated"):
        cache.check()
    host.fork([0], [2])
    host.same_tables(cache)
    cache.truncate([2, 2], [3, 1])
    with pytest.raises(RuntimeError, match="out of range or repeated"):
        cache.check()
    host.truncate([2], [3])
    host.same_tables(cache)


def test_copy_pages(cuda_device):
    cache = filled(cuda_device, 20, layers=3)
    host = R.HostCache.like(cache)
    cache.copy_pages([3, 4, 99, 5], [10, 19, 1, -1])
    host.pages[:, 10], host.pages[:, 19] = host.pages[:, 3], host.pages[:, 4]
    host.same(cache)
    cache.copy_pages([], [])
    host.same(cache)


def test_empty_calls(cuda_device):
    cache = make(cuda_device, [5])
    host = R.HostCache.like(cache)
    none = torch.empty(0, dtype=torch.int32, device=cuda_device)
    cache.extend(none, 3)
    cache.fork(none, none)
    cache.truncate(none, none)
    cache.free(none)
    assert cache.attention(torch.empty(0, 2, 4, 128, dtype=torch.half, device=cuda_device), seqs=none).numel() == 0
    assert cache.attention(torch.empty(1, 0, 4, 128, dtype=torch.half, device=cuda_device), seqs=[0]).numel() == 0
    assert cache.read([0], tokens=0)[0].shape == (1, 0, 2, 128)
    cache.write(torch.empty(1, 0, 2, 128, device=cuda_device), torch.empty(1, 0, 2, 128, device=cuda_device), seqs=[0])
    cache.check()
    host.same(cache)


def test_extend_adds_pages_up_in_64_bits(cuda_device):
    """32 sequences that ask for 2^30 tokens each: 2^31 pages, which 32 bits would take for none."""
    cache = Kv4Cache(64, kv_heads=1, max_seqs=32, max_tokens=1 << 30, page_size=16, dim_group_size=128,
                     device=cuda_device)
    seqs = torch.arange(32, dtype=torch.int32, device=cuda_device)
    cache.extend(seqs, 1 << 30)
    with pytest.raises(RuntimeError, match="too few free pages"):
        cache.check()
    assert cache.free_pages() == 64 and not cache.lengths.any()
    assert int(cache.table.min()) == -1 == int(cache.table.max())
    cache.extend(seqs, 17)
    cache.check()
    assert cache.free_pages() == 0 and cache.table[:, :2].flatten().tolist() == list(range(64))


def test_nothing_is_written_after_a_failed_extend(cuda_device):
    """Branches of a pool too full for their copies: the shared page keeps its bytes, and the step can be repeated."""
    cache = filled(cuda_device, 4)
    cache.extend([0], 40)
    cache.fork([0, 0], [1, 2])
    cache.check()
    host = R.HostCache.like(cache)
    x = torch.randn(2, 2, 1, 2, 128, generator=torch.Generator().manual_seed(1))
    keys, values = x.to(cuda_device)
    cache.extend([1, 2], 1)  # two copies, one free page
    for layer in range(2):
        cache.write(keys, values, seqs=[1, 2], layer=layer)
    cache.extend([1], 1)  # would fit, but a step that failed is not known yet
    for layer in range(2):
        cache.write(keys[:1], values[:1], seqs=[1], layer=layer)
    host.same(cache)
    cache.free([2])
    host.truncate([2], [0])
    with pytest.raises(RuntimeError, match="too few free pages"):
        cache.check()
    host.same(cache)
    assert host.extend([1], [1])
    cache.extend([1], 1)
    for layer in range(2):
        cache.write(keys[:1], values[:1], seqs=[1], layer=layer)
        for h in range(2):
            host.put(layer, 1, h, 40, x[0, 0, 0, h].numpy(), x[1, 0, 0, h].numpy())
    cache.check()
    host.same(cache)


def test_other_errors_do_not_hold_writes_back(cuda_device):
    cache = filled(cuda_device, 8)
    cache.extend([0, 0, 77], 20)
    host = R.HostCache.like(cache)
    x = torch.randn(1, 20, 2, 128, generator=torch.Generator().manual_seed(2))
    cache.write(x.to(cuda_device), -x.to(cuda_device), seqs=[0])
    for t in range(20):
        for h in range(2):
            host.put(0, 0, h, t, x[0, t, h].numpy(), -x[0, t, h].numpy())
    host.same(cache)
    with pytest.raises(RuntimeError, match="out of range or repeated"):
        cache.check()


def test_64_bit_ids_and_lengths_do_not_wrap(cuda_device):
    """int64 arguments past 32 bits: a length above every sequence's, an id and a count out of range."""
    def wide(*values):
        return torch.tensor(values, dtype=torch.int64, device=cuda_device)

    cache = filled(cuda_device, 20)
    cache.extend([0, 1], 20)
    host = R.HostCache.like(cache)
    cache.truncate([0, 1], wide(2 ** 63 - 1, 2 ** 32))
    cache.check()
    host.same(cache)
    for call in (lambda: cache.free(wide(2 ** 32)), lambda: cache.truncate(wide(2 ** 32 + 1), [3]),
                 lambda: cache.fork(wide(0), wide(2 ** 32 + 1)), lambda: cache.fork(wide(2 ** 32), wide(2)),
                 lambda: cache.extend(wide(-2 ** 32), 1)):
        call()
        with pytest.raises(RuntimeError, match="out of range or repeated"):
            cache.check()
        host.same(cache)
    cache.extend([0, 1], wide(2 ** 32, 2 ** 62))
    with pytest.raises(RuntimeError, match="table columns"):
        cache.check()
    host.same(cache)
    cache.truncate([0], wide(-2 ** 63))
    cache.check()
    host.truncate([0], [0])
    host.same(cache)


def test_strides_of_axes_with_one_entry_do_not_matter(cuda_device):
    """Rows that start on 16 bytes, in views whose axes of size 1 have odd strides."""
    cache = make(cuda_device, [40], kv_heads=2, page=16)
    wide = random_queries((1, 3 * 1028), torch.float16, cuda_device, 5)
    plain = wide[:, :1024].clone().view(1, 8, 128)
    want = cache.attention(plain, seqs=[0])
    index = torch.arange(30, device=cuda_device).expand(1, 8, 30)
    picked = cache.attention_selected(plain, index, seqs=[0])
    one = torch.as_strided(wide, (1, 8, 128), (1028, 128, 1))
    assert torch.equal(cache.attention(one, seqs=[0]), want)
    assert torch.equal(cache.attention_selected(one, index, seqs=[0]), picked)
    token = torch.as_strided(wide, (1, 1, 8, 128), (1028, 13, 128, 1))
    assert torch.equal(cache.attention(token, seqs=[0])[:, 0], want)
    few = make(cuda_device, [40], kv_heads=1, page=16)
    head = torch.as_strided(wide, (1, 2, 1, 128), (3, 1024, 129, 1))
    assert torch.equal(few.attention(head, seqs=[0]), few.attention(head.clone(), seqs=[0]))
    odd = torch.as_strided(wide, (1, 2, 1, 128), (3, 1028, 129, 1))  # here the second token's row is not aligned
    assert torch.equal(few.attention(odd, seqs=[0]), few.attention(odd.clone(), seqs=[0]))


def test_attention_of_logits_far_below_zero(cuda_device):
    """bf16 queries whose every logit is below -1e30: a token is seen however small its logit."""
    cache = Kv4Cache(8, kv_heads=1, max_seqs=1, max_tokens=100, page_size=16, device=cuda_device)
    cache.extend([0], 70)
    values = torch.randn(1, 70, 1, 128, generator=torch.Generator().manual_seed(1))
    keys = torch.ones(1, 70, 1, 128)
    keys[0, 50:] = 1.25
    cache.write(keys.to(cuda_device), values.to(cuda_device), seqs=[0])
    queries = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16, device=cuda_device)
    queries[0, 0, 0] = -1e30
    queries[0, 0, 1] = -1e32
    queries[0, 0, 2] = -3e34
    queries[0, 0, 3] = 1e32
    host = R.HostCache.like(cache)
    v = np.stack([host.get(0, 0, 0, t)[1] for t in range(70)])
    want = np.stack([v[:50].mean(0), v[:50].mean(0), v[:50].mean(0), v[50:].mean(0)])[None, None]
    close(cache.attention(queries, seqs=[0]), want, np.abs(v).max())
    picked = torch.arange(70, device=cuda_device).expand(1, 4, 70)
    close(cache.attention_selected(queries[:, 0], picked, seqs=[0]), want[:, 0], np.abs(v).max())


def test_one_workspace_for_calls_of_several_sizes(cuda_device):
    """A workspace of the largest call serves smaller ones in turn, of either attention."""
    lengths = [(211 * i) % 1500 for i in range(40)]
    cache = make(cuda_device, lengths, kv_heads=2, page=16)
    workspace = cache.workspace(40, 16, 5)
    calls = []
    for n, heads, q_len in ((40, 16, 5), (1, 2, 1), (7, 8, 1), (40, 16, 1), (3, 8, 4), (1, 16, 5)):
        seqs = torch.arange(40 - n, 40, dtype=torch.int32, device=cuda_device)
        q = random_queries((n, q_len, heads, 128), torch.float16, cuda_device, n + heads)
        calls.append((cache.attention, (q,), seqs))
        index = torch.randint(0, 1500, (n, heads, 70), generator=torch.Generator().manual_seed(n)).to(cuda_device)
        calls.append((cache.attention_selected, (q[:, 0], index), seqs))
    want = [call(*args, seqs=seqs) for call, args, seqs in calls]
    for _ in range(3):
        for (call, args, seqs), out in zip(calls, want):
            assert torch.equal(call(*args, seqs=seqs, workspace=workspace), out)
    with pytest.raises(RuntimeError, match="workspace"):
        cache.attention(random_queries((1, 1, 2, 128), torch.float16, cuda_device, 0), seqs=[0],
                        workspace=workspace[:1 << 16])
    with pytest.raises(ValueError, match="workspace"):
        cache.attention(random_queries((1, 1, 2, 128), torch.float16, cuda_device, 0), seqs=[0],
                        workspace=workspace.int())


def test_page_operations_and_selected_attention_in_a_graph(cuda_device):
    """fork, extend, write, attention_selected, truncate, free and compact captured once and replayed."""
    cache, twin = (make(cuda_device, [37, 50], kv_heads=2, page=16, spare=12, max_seqs=5) for _ in range(2))
    x = torch.randn(3, 4, 8, 128, generator=torch.Generator().manual_seed(3)).half().to(cuda_device)
    q, k, v = x[0], x[1, :, :2].contiguous(), x[2, :, :2].contiguous()
    ids = {name: torch.tensor(value, dtype=torch.int32, device=cuda_device) for name, value in {
        "parents": [0, 1, 0], "children": [2, 3, 4], "all": [0, 2, 3, 4], "some": [2, 0], "kept": [30, 38],
        "gone": [3, 4]}.items()}
    index = torch.randint(0, 60, (4, 8, 40), generator=torch.Generator().manual_seed(4)).to(cuda_device)
    workspaces = {id(c): c.workspace(4, 8) for c in (cache, twin)}

    def step(c):
        c.fork(ids["parents"], ids["children"])
        c.extend(ids["all"], 1)
        c.write(k, v, seqs=ids["all"])
        out = c.attention_selected(q, index, seqs=ids["all"], workspace=workspaces[id(c)])
        whole = c.attention(q, seqs=ids["all"], workspace=workspaces[id(c)])
        c.truncate(ids["some"], ids["kept"])
        c.free(ids["gone"])
        c.compact()
        return out, whole

    snapshot = cache.tables.clone(), cache.pages.clone()
    step(cache)
    cache.tables.copy_(snapshot[0])
    cache.pages.copy_(snapshot[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(4):
        k.copy_(x[1, :, :2] * (i + 1))
        graph.replay()
        want = step(twin)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(cache.tables, twin.tables) and torch.equal(cache.pages, twin.pages)
        assert torch.equal(cache.status[1:3], twin.status[1:3])
    cache.check()
    twin.check()
    del graph


def test_page_operations_on_thousands_of_sequences(cuda_device):
    """More entries than the plans' threads, and tables that a fork takes two launches for."""
    rng = np.random.default_rng(5)
    cache = Kv4Cache(14000, kv_heads=1, max_seqs=3000, max_tokens=20 * 16, page_size=16, dim_group_size=128,
                     device=cuda_device)
    cache.pages.random_(0, 256)
    host = R.HostCache.like(cache)

    def ids(values):
        return torch.tensor(values, dtype=torch.int32, device=cuda_device)

    def extend(seqs, counts):
        assert host.extend(seqs, counts)
        cache.extend(ids(seqs), ids(counts))
        cache.check()
        host.same(cache)

    extend(rng.permutation(3000).tolist(), rng.integers(0, 40, 3000).tolist())
    for n in (1400, 2000):
        parents, children = rng.integers(0, 3000, n).tolist(), rng.permutation(3000)[:n].tolist()
        host.fork(parents, children)
        cache.fork(ids(parents), ids(children))
        host.same(cache)
        extend(rng.permutation(3000)[:2900].tolist(), rng.integers(0, 4, 2900).tolist())
    some, lengths = rng.permutation(3000).tolist(), rng.integers(-5, 50, 3000).tolist()
    host.truncate(some, lengths)
    cache.truncate(ids(some), ids(lengths))
    host.truncate(some[:1100], [0] * 1100)
    cache.free(ids(some[:1100]))
    host.same(cache)
    assert cache.status[0].item() == 0
    cache.compact()
    assert tuple(cache.status[1:3].tolist()) == host.compact()
    host.same(cache)
    before = host.refs.copy()
    assert not host.extend(some, [310 - int(host.lengths[s]) for s in some])
    cache.extend(ids(some), ids([310 - int(host.lengths[s]) for s in some]))
    with pytest.raises(RuntimeError, match="too few free pages"):
        cache.check()
    assert np.array_equal(before, host.refs)
    host.same(cache)


@pytest.mark.parametrize("heads,group,dtype", [(12, 32, torch.bfloat16), (9, 64, torch.float16),
                                               (16, 128, torch.float32)])
def test_rows_and_attention_of_many_heads(cuda_device, heads, group, dtype):
    """More KV heads than a block has warps."""
    cache = make(cuda_device, [37, 20], kv_heads=heads, page=16, group=group)
    host = R.HostCache.like(cache)
    x = torch.randn(2, 2, 7, heads, 128, generator=torch.Generator().manual_seed(heads)).to(dtype)
    cache.write(x[0].to(cuda_device), x[1].to(cuda_device), seqs=[0, 1])
    for s, length in enumerate((37, 20)):
        for t in range(7):
            for h in range(heads):
                host.put(0, s, h, length - 7 + t, x[0, s, t, h].float().numpy(), x[1, s, t, h].float().numpy())
    host.same(cache)
    got = cache.read([1, 0], tokens=40, dtype=dtype)
    for which in range(2):
        want = np.zeros((2, 40, heads, 128))
        for i, s in enumerate((1, 0)):
            for t in range((37, 20)[s]):
                for h in range(heads):
                    want[i, t, h] = host.get(0, s, h, t)[which]
        assert torch.equal(got[which].cpu(), torch.from_numpy(want).float().to(dtype))
    queries = random_queries((2, 3, 2 * heads, 128), torch.float16, cuda_device, heads)
    want, most = expect(cache, host, queries, lambda at: (at[0], range((37, 20)[at[0]] - 3 + at[1] + 1)))
    close(cache.attention(queries, seqs=[0, 1]), want, most)


# -- refusals -----------------------------------------------------------------------
def test_refusals(cuda_device):
    cache = make(cuda_device, [5, 6])
    x = torch.randn(2, 3, 2, 128, device=cuda_device)
    q = torch.randn(2, 3, 4, 128, device=cuda_device).half()
    with pytest.raises(ValueError, match="keys and values must be"):
        cache.write(x[..., :64], x[..., :64], seqs=[0, 1])
    with pytest.raises(ValueError, match="keys and values must be"):
        cache.write(x, x[:, :2], seqs=[0, 1])
    with pytest.raises(RuntimeError, match="share an fp32/fp16/bf16"):
        cache.write(x, x.half(), seqs=[0, 1])
    with pytest.raises(RuntimeError, match="share an fp32/fp16/bf16"):
        cache.write(x.double(), x.double(), seqs=[0, 1])
    with pytest.raises(RuntimeError, match="cache's device"):
        cache.write(x.cpu(), x.cpu(), seqs=[0, 1])
    with pytest.raises(ValueError, match="layer must be"):
        cache.write(x, x, seqs=[0, 1], layer=1)
    with pytest.raises(ValueError, match="one value per listed sequence"):
        cache.write(x, x, seqs=[0, 1], counts=[1])
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        cache.attention(q.float(), seqs=[0, 1])
    with pytest.raises(ValueError, match="multiple of the cache's KV heads"):
        cache.attention(q[:, :, :3], seqs=[0, 1])
    with pytest.raises(ValueError, match="queries must be"):
        cache.attention(q, seqs=[0])
    with pytest.raises(ValueError, match="queries must be"):
        cache.attention(q[0, 0], seqs=[0])
    with pytest.raises(RuntimeError, match="cache's device"):
        cache.attention(q.cpu(), seqs=[0, 1])
    with pytest.raises(RuntimeError, match="seqs must be on the cache's device"):
        cache.attention(q, seqs=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32 or int64"):
        cache.attention(q, seqs=torch.zeros(2, device=cuda_device))
    index = torch.zeros(2, 4, 5, dtype=torch.int64, device=cuda_device)
    with pytest.raises(ValueError, match="indices must be"):
        cache.attention_selected(q[:, 0], index[:, :3], seqs=[0, 1])
    with pytest.raises(ValueError, match="int64"):
        cache.attention_selected(q[:, 0], index.int(), seqs=[0, 1])
    with pytest.raises(ValueError, match="valid mask"):
        cache.attention_selected(q[:, 0], index, seqs=[0, 1], valid_mask=index[..., :2] > 0)
    with pytest.raises(ValueError, match="bool or uint8"):
        cache.attention_selected(q[:, 0], index, seqs=[0, 1], valid_mask=index)
    with pytest.raises(ValueError, match="must not be negative"):
        cache.extend([0], -1)
    with pytest.raises(ValueError, match="same length"):
        cache.fork([0, 1], [0])
    with pytest.raises(ValueError, match="at most 4096"):
        cache.extend(list(range(5000)), 1)
    with pytest.raises(ValueError, match="must not be negative"):
        cache.read([0], start=-1, tokens=2)
    with pytest.raises(RuntimeError, match="fp32/fp16/bf16"):
        cache.read([0], tokens=2, dtype=torch.int8)
