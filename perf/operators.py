"""Cases of the 4-bit paged KV cache and of drafted-token verification, for timing and comparison.

Each case names one operator call (or the short sequence of calls that one decode
step makes) and its sizes.  ``run`` computes it in plain torch operations, in 32
bits and rounded once at the end, or, with ``own`` set, through the package's
entry points (``popkv_b200.kv4.Kv4Cache``, ``popkv_b200.speculative``).

The cache, as both forms hold it:

* ``pages``  uint8 [layers, num_pages, kv_heads, page_bytes].  The bytes of a
  (page, head) are ``page_size / 16`` tiles of 16 tokens; a tile is 16 x 64 bytes
  of 4-bit keys, 16 x 64 bytes of 4-bit values, then per token the fp16 pairs
  (low, delta) of the key groups and of the value groups, ``128 / G`` each.  A
  number n in 0..15 of a group of G dims stands for low + n * delta.
* key bytes: natural byte b holds dim 2b (low nibble) and 2b + 1; the 16 words of
  a row (4 bytes each), as a 4 x 4 matrix, are stored transposed.  Value bytes: the
  64 natural bytes of a row, as an 8 x 8 matrix, are stored transposed.
* ``tables`` int32, one buffer: refs [num_pages] (0: free page), lengths [max_seqs],
  table [max_seqs, max_pages] (the page of each ``page_size`` tokens, -1 past the end).
"""
import math
import random

import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LIMIT = 65504.0  # the largest fp16 value


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    heads = {"q_heads": 32, "kv_heads": 8}
    return [
        # One decode step of 64 sequences: a token each enters the cache and is read back.
        {"name": "write 64x1", "op": "write", "n": 64, "tokens": 1, "prior": 1000, "dims": 32, "page": 64,
         "dtype": "bf16", **heads},
        # A prefill chunk of one long prompt, an odd number of tokens at an odd offset.
        {"name": "write 1x8191", "op": "write", "n": 1, "tokens": 8191, "prior": 8195, "dims": 32, "page": 64,
         "dtype": "bf16", **heads},
        # The first tokens of a short chat: latency only.
        {"name": "attend 1x77", "op": "attend", "n": 1, "shortest": 77, "longest": 77, "q_len": 1, "ragged": False,
         "dims": 32, "page": 64, "dtype": "bf16", **heads},
        # The dense layers of a single long sequence's decode step.
        {"name": "attend 1x32768", "op": "attend", "n": 1, "shortest": 32768, "longest": 32768, "q_len": 1,
         "ragged": False, "dims": 32, "page": 64, "dtype": "bf16", **heads},
        # A serving batch of very different lengths, one slot empty.
        {"name": "attend 33 ragged", "op": "attend", "n": 33, "shortest": 0, "longest": 8192, "q_len": 1,
         "ragged": False, "dims": 64, "page": 16, "dtype": "fp16", **heads},
        # Four drafted tokens and the last accepted one, checked against long contexts; drafts of uneven length.
        {"name": "attend 4x131072 drafts", "op": "attend", "n": 4, "shortest": 131000, "longest": 131072, "q_len": 5,
         "ragged": True, "dims": 32, "page": 64, "dtype": "bf16", **heads},
        # The sparse layers of a single sequence: the budget's tokens of each query head.
        {"name": "select 4096 of 32768", "op": "select", "n": 1, "longest": 32768, "budget": 4096, "masked": False,
         "dims": 32, "page": 64, "dtype": "bf16", **heads},
        # The same for a batch of long sequences, with slots masked out.
        {"name": "select 8x4096 of 131072", "op": "select", "n": 8, "longest": 131072, "budget": 4096, "masked": True,
         "dims": 32, "page": 64, "dtype": "bf16", **heads},
        # A prompt branched into parallel samples, each of which then writes one token.
        {"name": "fork 1 to 8", "op": "fork", "parents": 1, "branches": 8, "prefix": 4001, "tokens": 1, "layers": 32,
         "kv_heads": 8, "dims": 32, "page": 64},
        # A pool with holes after half of its sequences ended, moved together.
        {"name": "compact 32 layers", "op": "compact", "seqs": 40, "longest": 1920, "keep": 0.5, "layers": 32,
         "kv_heads": 8, "dims": 32, "page": 64},
        # One sequence's drafted tokens: latency only.
        {"name": "verify 1x4", "op": "verify", "n": 1, "drafts": 4, "vocab": 128256, "dtype": "fp32",
         "proposal": True, "ragged": False},
        # A serving batch's, drafts of uneven length.
        {"name": "verify 64x8", "op": "verify", "n": 64, "drafts": 8, "vocab": 128256, "dtype": "fp32",
         "proposal": True, "ragged": True},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("write", "attend", "attend", "select", "fork", "compact", "verify", "verify"))
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"op": op}
    if op != "verify":
        case.update(kv_heads=kv_heads, dims=rng.choice((32, 64, 128)), page=rng.choice((16, 32, 64, 128)))
    if op in ("write", "attend", "select"):
        case.update(q_heads=kv_heads * rng.choice((1, 2, 4, 4, 7, 8)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    if op == "write":
        case.update(n=_spread(rng, 1, 64), prior=_spread(rng, 1, 4096) - 1, dtype=rng.choice(("bf16", "fp16", "fp32")))
        case["tokens"] = _spread(rng, 1, max(1, 8192 // case["n"]))
    elif op == "attend":
        case["n"] = _spread(rng, 1, 64)
        case["longest"] = _spread(rng, 1, min(131072, 262144 // case["n"]))
        case["shortest"] = rng.choice((0, case["longest"] // 2, case["longest"]))
        case["q_len"] = rng.choice((1, 1, 1, 2, 3, 5, 8))
        case["ragged"] = rng.random() < 0.5
    elif op == "select":
        case["n"] = _spread(rng, 1, 16)
        case["longest"] = _spread(rng, 64, min(131072, 524288 // case["n"]))
        case["budget"] = _spread(rng, 1, min(4096, case["longest"], (1 << 20) // (case["n"] * case["q_heads"])))
        case["masked"] = rng.random() < 0.5
    elif op == "fork":
        case.update(parents=_spread(rng, 1, 8), branches=_spread(rng, 1, 8), prefix=_spread(rng, 1, 8192),
                    tokens=_spread(rng, 1, 32), layers=rng.choice((1, 2, 16)))
    elif op == "compact":
        case.update(seqs=_spread(rng, 2, 64), longest=_spread(rng, 64, 2048), keep=round(rng.uniform(0.2, 0.9), 3),
                    layers=rng.choice((1, 2, 16)))
    else:
        case.update(n=_spread(rng, 1, 64), drafts=rng.randint(1, 8), vocab=_spread(rng, 1000, 128256),
                    dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), proposal=rng.random() < 0.75,
                    ragged=rng.random() < 0.5)
    return case


def _lengths(case):
    """Cached tokens of each sequence: spread evenly over the case's range, in a mixed order."""
    n, low, high = case["n"], case.get("shortest", case["longest"]), case["longest"]
    if n == 1:
        return [high]
    order = [7 * i % n if n % 7 else i for i in range(n)]
    return [low + (high - low) * i // (n - 1) for i in order]


def _counts(case, most):
    """Query or draft tokens of each sequence."""
    return [1 + (5 * i + most - 1) % most if case["ragged"] else most for i in range(case["n"])]


def _kept(case):
    """Lengths of the pool's sequences, and whether each is still there (a fixed choice of the case)."""
    rng = random.Random(case["seqs"] * 1000003 + case["longest"])
    lengths = [rng.randint(max(1, case["longest"] // 4), case["longest"]) for _ in range(case["seqs"])]
    order = rng.sample(range(case["seqs"]), case["seqs"])
    keep = max(1, round(case["keep"] * case["seqs"]))
    return lengths, [order[i] < keep for i in range(case["seqs"])]


def _pages_of(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------------------
# The plain cache
# ---------------------------------------------------------------------------
def _page_bytes(case):
    return case["page"] * (D + 8 * (D // case["dims"]))


def _quantise(x, dims):
    """Whole numbers 0..15 [..., D] and their fp16 (low, delta) [..., D / dims] of values x."""
    x = torch.nan_to_num(x.float(), nan=0.0).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, dims))
    low = x.amin(-1).half()
    delta = ((x.amax(-1) - low.float()) / 15).clamp_min(0).half()
    scale = torch.where(delta > 0, 1 / delta.float(), 0.0)
    n = ((x - low.float()[..., None]) * scale[..., None]).round().clamp(0, 15).to(torch.uint8)
    return n.flatten(-2), low, delta


def _natural_bytes(n):
    return n[..., 0::2] | n[..., 1::2] << 4


def _stored_keys(n):
    return _natural_bytes(n).unflatten(-1, (4, 4, 4)).transpose(-3, -2).flatten(-3)


def _stored_values(n):
    return _natural_bytes(n).unflatten(-1, (8, 8)).transpose(-2, -1).flatten(-2)


def _stored_pairs(k_low, k_delta, v_low, v_delta):
    pairs = torch.cat([torch.stack([k_low, k_delta], -1), torch.stack([v_low, v_delta], -1)], -2)
    return pairs.flatten(-2).contiguous().view(torch.uint8)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _plain_rows(rows, dims):
    """fp32 keys and values [..., D] of stored (key bytes, value bytes, pair bytes)."""
    kb, vb, pairs = rows
    kn = _nibbles(kb.unflatten(-1, (4, 4, 4)).transpose(-3, -2).flatten(-3))
    vn = _nibbles(vb.unflatten(-1, (8, 8)).transpose(-2, -1).flatten(-2))
    pairs = pairs.contiguous().view(torch.float16).unflatten(-1, (2, D // dims, 2)).float()

    def values(n, p):
        return (p[..., 0, None] + n.unflatten(-1, (-1, dims)) * p[..., 1, None]).flatten(-2)

    return values(kn, pairs[..., 0, :, :]), values(vn, pairs[..., 1, :, :])


def _parts(pages, case):
    """The key, value and pair bytes of pages [..., page_bytes], each [..., tiles, 16, bytes]."""
    tiles = pages.unflatten(-1, (case["page"] // 16, -1))
    return (tiles[..., :1024].unflatten(-1, (16, 64)), tiles[..., 1024:2048].unflatten(-1, (16, 64)),
            tiles[..., 2048:].unflatten(-1, (16, -1)))


def _views(state):
    """refs, lengths and table of the state's table buffer."""
    p, s = state["num_pages"], state["max_seqs"]
    t = state["tables"]
    return t[:p], t[p:p + s], t[p + s:].view(s, state["max_pages"])


def _rows_at(state, seqs, heads, positions, layer=0):
    """Stored rows of tokens ``positions`` [n, ...] of heads ``heads`` (broadcastable) of sequences ``seqs``."""
    case = state["case"]
    _, _, table = _views(state)
    size = case["page"]
    lead = seqs.view(-1, *[1] * (positions.dim() - 1)).long()
    page = table[lead, (positions // size).clamp(0, state["max_pages"] - 1)].long().clamp_min(0)
    row = positions % size
    return [p[page, heads, row // 16, row % 16] for p in _parts(state["pages"][layer], case)]


def _empty_state(case, device, *, layers, num_pages, max_seqs, max_pages):
    shape = (layers, num_pages, case["kv_heads"], _page_bytes(case))
    return {"case": case, "num_pages": num_pages, "max_seqs": max_seqs, "max_pages": max_pages,
            "pages": torch.zeros(shape, dtype=torch.uint8, device=device),
            "tables": torch.cat([torch.zeros(num_pages + max_seqs, dtype=torch.int32, device=device),
                                 torch.full((max_seqs * max_pages,), -1, dtype=torch.int32, device=device)])}


def _give_pages(state, lengths, gen):
    """Hand the sequences pages in a random order of the pool."""
    refs, lens, table = _views(state)
    need = [_pages_of(t, state["case"]["page"]) for t in lengths]
    order = torch.randperm(state["num_pages"], device=refs.device, generator=gen).int()
    at = 0
    for s, count in enumerate(need):
        table[s, :count] = order[at:at + count]
        at += count
    refs[order[:at].long()] = 1
    lens[:len(lengths)] = torch.tensor(lengths, dtype=torch.int32, device=refs.device)


def _fill(state, gen):
    """Every page with quantised keys (outlier channels) and values, a few pages at a time."""
    case, heads = state["case"], state["case"]["kv_heads"]
    device = state["pages"].device
    factors = torch.randn((heads, 1, 1, D), device=device, generator=gen).mul(0.5).exp()
    step = max(1, (1 << 20) // (heads * case["page"]))
    for layer in state["pages"]:
        for at in range(0, state["num_pages"], step):
            part = layer[at:at + step]
            shape = (part.shape[0], heads, case["page"] // 16, 16, D)
            kn, kl, kd = _quantise(torch.randn(shape, device=device, generator=gen) * factors, case["dims"])
            vn, vl, vd = _quantise(torch.randn(shape, device=device, generator=gen), case["dims"])
            for to, rows in zip(_parts(part, case), (_stored_keys(kn), _stored_values(vn),
                                                     _stored_pairs(kl, kd, vl, vd))):
                to.copy_(rows)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    device = torch.device("cuda", 0)
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    state = globals()["_prepare_" + case["op"]](case, device, gen)
    if own and case["op"] != "verify":
        from popkv_b200.kv4 import Kv4Cache
        state["cache"] = Kv4Cache.from_tensors(state["pages"], state["tables"], max_seqs=state["max_seqs"],
                                               page_size=case["page"], dim_group_size=case["dims"])
    return state


def _normal(shape, gen, dtype):
    return torch.randn(shape, device=gen.device, generator=gen).to(dtype)


def _prepare_write(case, device, gen):
    total = case["prior"] + case["tokens"]
    per = _pages_of(total, case["page"])
    state = _empty_state(case, device, layers=1, num_pages=case["n"] * per + 3, max_seqs=case["n"], max_pages=per)
    _give_pages(state, [total] * case["n"], gen)
    qh, kh = case["q_heads"], case["kv_heads"]
    qkv = _normal((case["n"], case["tokens"], qh + 2 * kh, D), gen, DTYPES[case["dtype"]])
    qkv[:, :, qh:qh + kh] *= torch.randn((kh, D), device=device, generator=gen).mul(0.5).exp().to(qkv.dtype)
    state.update(seqs=torch.arange(case["n"], dtype=torch.int32, device=device),
                 keys=qkv[:, :, qh:qh + kh], values=qkv[:, :, qh + kh:])
    return state


def _prepare_attend(case, device, gen):
    lengths = _lengths(case)
    counts = [min(c, t) for c, t in zip(_counts(case, case["q_len"]), lengths)]
    need = sum(_pages_of(t, case["page"]) for t in lengths)
    state = _empty_state(case, device, layers=1, num_pages=need + 5, max_seqs=case["n"] + 1,
                         max_pages=max(1, _pages_of(max(lengths), case["page"])))
    _give_pages(state, lengths, gen)
    _fill(state, gen)
    state.update(seqs=torch.randperm(case["n"], device=device, generator=gen).int(),
                 queries=_normal((case["n"], case["q_len"], case["q_heads"], D), gen, DTYPES[case["dtype"]]))
    state["counts"] = torch.tensor(counts, dtype=torch.int32, device=device)[state["seqs"].long()]
    return state


def _prepare_select(case, device, gen):
    n, tokens = case["n"], case["longest"]
    per = _pages_of(tokens, case["page"])
    state = _empty_state(case, device, layers=1, num_pages=n * per + 5, max_seqs=n, max_pages=per)
    _give_pages(state, [tokens] * n, gen)
    _fill(state, gen)
    scores = torch.rand((n, case["q_heads"], tokens), device=device, generator=gen)
    scores[..., -1] = 2.0  # the current token is always among them
    indices = scores.topk(case["budget"]).indices.sort().values
    valid = None
    if case["masked"]:
        valid = torch.rand(indices.shape, device=device, generator=gen) < 0.9
        valid[0, 0] = False
    state.update(seqs=torch.arange(n, dtype=torch.int32, device=device), indices=indices, valid=valid,
                 queries=_normal((n, case["q_heads"], D), gen, DTYPES[case["dtype"]]))
    return state


def _prepare_fork(case, device, gen):
    p, b = case["parents"], case["branches"]
    total = case["prefix"] + case["tokens"]
    per = _pages_of(total, case["page"])
    extra = per - case["prefix"] // case["page"]
    state = _empty_state(case, device, layers=case["layers"], num_pages=p * (_pages_of(case["prefix"], case["page"])
                         + b * extra) + 7, max_seqs=p * (1 + b) + 1, max_pages=per + 1)
    _give_pages(state, [case["prefix"]] * p, gen)
    state["pages"].random_(0, 256, generator=gen)
    parents = torch.arange(p, dtype=torch.int32, device=device)
    state.update(parents=parents.repeat_interleave(b),
                 children=(p + torch.randperm(p * b, device=device, generator=gen)).int())
    return state


def _prepare_compact(case, device, gen):
    lengths, keep = _kept(case)
    per = max(_pages_of(t, case["page"]) for t in lengths)
    state = _empty_state(case, device, layers=case["layers"], num_pages=sum(_pages_of(t, case["page"])
                         for t in lengths), max_seqs=case["seqs"], max_pages=per)
    _give_pages(state, lengths, gen)
    refs, lens, table = _views(state)
    gone = ~torch.tensor(keep, device=device)
    refs[table[gone][table[gone] >= 0].long()] = 0
    table[gone], lens[gone] = -1, 0
    state["pages"].random_(0, 256, generator=gen)
    state["tables_before"] = state["tables"].clone()
    return state


def _prepare_verify(case, device, gen):
    n, k, vocab, dtype = case["n"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.randn((n, k + 1, vocab), device=device, generator=gen) * 3
    target = logits.softmax(-1).to(dtype)
    logits = logits[:, :k] + torch.randn((n, k, vocab), device=device, generator=gen) * 0.7
    draft = logits.softmax(-1)
    race = draft / torch.empty_like(draft).exponential_(generator=gen)
    state = {"case": case, "target": target, "draft": draft.to(dtype) if case["proposal"] else None,
             "tokens": race.argmax(-1), "uniforms": torch.rand((n, k), device=device, generator=gen),
             "noise": torch.empty((n, vocab), device=device).exponential_(generator=gen), "counts": None}
    if case["ragged"]:
        counts = [c - 1 for c in _counts(case, k + 1)]
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device=device)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["op"]](state)


def _own_write(state):
    case, cache = state["case"], state["cache"]
    cache.write(state["keys"], state["values"], seqs=state["seqs"])
    return cache.read(state["seqs"], start=case["prior"], tokens=case["tokens"], dtype=state["keys"].dtype)


def _plain_write(state):
    case = state["case"]
    n, tokens, heads = case["n"], case["tokens"], case["kv_heads"]
    _, lengths, table = _views(state)
    device = table.device
    position = (lengths[state["seqs"].long()].long() - tokens)[:, None] + torch.arange(tokens, device=device)
    page = table[state["seqs"].long()[:, None], position // case["page"]].long()
    row = position % case["page"]
    head = torch.arange(heads, device=device)
    kn, kl, kd = _quantise(state["keys"], case["dims"])
    vn, vl, vd = _quantise(state["values"], case["dims"])
    at = (page[..., None], head, row[..., None] // 16, row[..., None] % 16)
    for to, rows in zip(_parts(state["pages"][0], case), (_stored_keys(kn), _stored_values(vn),
                                                          _stored_pairs(kl, kd, vl, vd))):
        to[at] = rows
    positions = (case["prior"] + torch.arange(tokens, device=device)).view(1, -1, 1).expand(n, -1, heads)
    keys, values = _plain_rows(_rows_at(state, state["seqs"], head, positions), case["dims"])
    return keys.to(state["keys"].dtype), values.to(state["keys"].dtype)


def _own_attend(state):
    return state["cache"].attention(state["queries"], seqs=state["seqs"], counts=state["counts"])


def _softmax_sum(logits, seen, values):
    """Softmax over the last axis of the seen logits (zeros where a row sees none), times values."""
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = (logits - torch.where(top > -math.inf, top, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p / torch.where(total > 0, total, 1.0), values)


def _plain_attend(state):
    case = state["case"]
    n, heads, q_len, q_heads = case["n"], case["kv_heads"], case["q_len"], case["q_heads"]
    _, lengths, table = _views(state)
    seqs = state["seqs"].long()
    pages = state["pages"][0][table[seqs].long().clamp_min(0)]  # [n, pages, heads, bytes]
    rows = [p.permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for p in _parts(pages, case)]
    keys, values = _plain_rows(rows, case["dims"])  # [n, heads, tokens, D]
    q = state["queries"].float().view(n, q_len, heads, -1, D).permute(0, 2, 1, 3, 4).reshape(n, heads, -1, D)
    logits = torch.matmul(q, keys.transpose(-2, -1)) / math.sqrt(D)
    row = torch.arange(q_len, device=q.device)
    counts = state["counts"].long()[:, None]
    last = torch.where(row < counts, lengths[seqs].long()[:, None] - counts + row, -1)  # [n, q_len]
    seen = torch.arange(keys.shape[2], device=q.device) <= last[:, :, None]
    seen = seen[:, None, :, None].expand(n, heads, q_len, q_heads // heads, -1).flatten(2, 3)
    out = _softmax_sum(logits, seen, values)
    out = out.view(n, heads, q_len, -1, D).permute(0, 2, 1, 3, 4).reshape(n, q_len, q_heads, D)
    return out.to(state["queries"].dtype)


def _own_select(state):
    return state["cache"].attention_selected(state["queries"], state["indices"], seqs=state["seqs"],
                                             valid_mask=state["valid"])


def _plain_select(state):
    case = state["case"]
    _, lengths, _ = _views(state)
    q_heads = case["q_heads"]
    head = (torch.arange(q_heads, device=state["indices"].device) // (q_heads // case["kv_heads"]))[:, None]
    keys, values = _plain_rows(_rows_at(state, state["seqs"], head, state["indices"]), case["dims"])
    logits = torch.matmul(keys, state["queries"].float()[..., None])[..., 0] / math.sqrt(D)
    seen = (state["indices"] >= 0) & (state["indices"] < lengths[state["seqs"].long()].view(-1, 1, 1))
    seen = seen if state["valid"] is None else seen & state["valid"]
    return _softmax_sum(logits[..., None, :], seen[..., None, :], values)[..., 0, :].to(state["queries"].dtype)


def _own_fork(state):
    cache = state["cache"]
    cache.fork(state["parents"], state["children"])
    cache.extend(state["children"], state["case"]["tokens"])
    return state["tables"], state["pages"]


def _plain_fork(state):
    size = state["case"]["page"]
    refs, lengths, table = _views(state)
    parents, children = state["parents"].long(), state["children"].long()
    # Share: children give their pages back and take their parents'.
    rows, before = table[parents], table[children]
    refs.index_add_(0, before.clamp_min(0).flatten().long(), -(before >= 0).int().flatten())
    refs.index_add_(0, rows.clamp_min(0).flatten().long(), (rows >= 0).int().flatten())
    table[children] = rows
    lengths[children] = lengths[parents]
    # Extend: new pages from the lowest free ones, a copy of a shared last page first.
    tokens = state["case"]["tokens"]
    held = lengths[children].long()
    old, new = (held + size - 1) // size, (held + tokens + size - 1) // size
    last = table[children, (old - 1).clamp_min(0)].long().clamp_min(0)
    copied = (held % size > 0) & (refs[last] > 1)
    need = new - old + copied.long()
    first = need.cumsum(0) - need
    free = torch.sort((refs != 0).to(torch.int8), stable=True).indices
    width = _pages_of(tokens, size) + 2
    j = torch.arange(width, device=refs.device)
    took = j < need[:, None]
    page = free[(first[:, None] + j).clamp_max(state["num_pages"] - 1)]
    column = (old - copied.long())[:, None] + j
    source = torch.where(copied, last, 0)
    target = torch.where(copied, page[:, 0], source)
    state["pages"][:, target] = state["pages"][:, source]
    refs.index_add_(0, last, -copied.int())
    row, at = took.nonzero(as_tuple=True)
    refs[page[row, at]] = 1
    table[children[row], column[row, at]] = page[row, at].int()
    lengths[children] += tokens
    return state["tables"], state["pages"]


def _own_compact(state):
    state["tables"].copy_(state["tables_before"])
    state["cache"].compact()
    return state["tables"], state["pages"]


def _plain_compact(state):
    state["tables"].copy_(state["tables_before"])
    refs, _, table = _views(state)
    live = refs > 0
    index = torch.arange(state["num_pages"], device=refs.device)
    below = index < live.sum()
    source, target = (live & ~below).nonzero()[:, 0], (~live & below).nonzero()[:, 0]
    state["pages"][:, target] = state["pages"][:, source]
    refs[target] = refs[source]
    refs[source] = 0
    place = index.index_put((source,), target).int()
    table.copy_(torch.where(table >= 0, place[table.clamp_min(0).long()], table))
    return state["tables"], state["pages"]


def _own_verify(state):
    from popkv_b200.speculative import verify_drafts
    return verify_drafts(state["target"], state["tokens"], state["uniforms"], state["noise"],
                         draft_probs=state["draft"], counts=state["counts"])


def _plain_verify(state):
    case, target, tokens = state["case"], state["target"], state["tokens"]
    n, k, vocab = case["n"], case["drafts"], case["vocab"]
    place = torch.arange(k + 1, device=tokens.device)
    counts = torch.full((n,), k, device=tokens.device) if state["counts"] is None else state["counts"].long()
    p = target[:, :k].gather(-1, tokens[..., None])[..., 0].float()
    q = torch.ones_like(p) if state["draft"] is None else state["draft"].gather(-1, tokens[..., None])[..., 0].float()
    agreed = (state["uniforms"] * q < p) & (place[:k] < counts[:, None])
    accepted = agreed.long().cumprod(-1).sum(-1)
    # The next token: from what the target has over the draft at the first refusal, from the target after the last.
    row = target[torch.arange(n, device=tokens.device), accepted].float()
    at = accepted.clamp_max(k - 1)
    refused = (accepted < counts)[:, None]
    drafted = tokens.gather(-1, at[:, None])
    if state["draft"] is None:
        over = row.scatter(-1, drafted, 0.0)
    else:
        over = (row - state["draft"][torch.arange(n, device=tokens.device), at].float()).clamp_min(0)
    refused = refused & (over > 0).any(-1, keepdim=True)
    weight = torch.where(refused, over, row)
    following = torch.where(weight > 0, weight / state["noise"], -1.0).argmax(-1)
    padded = torch.cat([tokens, tokens[:, :1]], -1)
    out = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None],
                                                                     following[:, None], -1))
    return out, accepted.int()


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact values
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    row = D + 8 * (D // case["dims"]) if op != "verify" else 0  # bytes of a cached token of one head
    if op == "write":
        rows = case["n"] * case["tokens"] * case["kv_heads"]
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": rows * (2 * 2 * D * size + 2 * row), "flops": rows * 2 * D * 6}
    if op == "attend":
        lengths = _lengths(case)
        io = 2 * case["n"] * case["q_len"] * case["q_heads"] * D * 2
        return {"bytes": sum(lengths) * case["kv_heads"] * row + io,
                "flops": 4 * D * case["q_heads"] * sum(t * min(c, t) for t, c in
                                                       zip(lengths, _counts(case, case["q_len"])))}
    if op == "select":
        slots = case["n"] * case["q_heads"] * case["budget"]
        return {"bytes": slots * (row + 8 + bool(case["masked"])) + 2 * case["n"] * case["q_heads"] * D * 2,
                "flops": slots * 4 * D}
    if op == "fork":
        m = case["parents"] * case["branches"]
        held = _pages_of(case["prefix"], case["page"])
        copies = m if case["prefix"] % case["page"] else 0
        page = case["layers"] * case["kv_heads"] * case["page"] * row
        return {"bytes": copies * 2 * page + m * held * 16, "flops": 0}
    if op == "compact":
        lengths, keep = _kept(case)
        total = sum(_pages_of(t, case["page"]) for t in lengths)
        live = sum(_pages_of(t, case["page"]) for t, k in zip(lengths, keep) if k)
        moved = live * (total - live) / total  # of live pages in a random order, those past the first `live`
        page = case["layers"] * case["kv_heads"] * case["page"] * row
        return {"bytes": moved * 2 * page + total * 12, "flops": 0}
    rows = 2 + bool(case["proposal"])
    size = DTYPES[case["dtype"]].itemsize
    return {"bytes": case["n"] * case["vocab"] * (size * (rows - 1) + 4), "flops": case["n"] * case["vocab"] * 2}


def exact(case, seed):
    if case["op"] == "write":
        state = prepare(case, seed)
        return _exact_stored(state["keys"], case["dims"]), _exact_stored(state["values"], case["dims"])
    if case["op"] in ("attend", "select"):
        return globals()["_exact_" + case["op"]](prepare(case, seed))
    return None  # whole numbers and bytes only


def _exact_stored(x, dims):
    """The nearest of the 16 values between a group's ends, in 64 bits (low and delta in fp16, as stored)."""
    shape = x.shape
    x = x.double().reshape(*shape[:-1], D // dims, dims)
    low = x.min(-1, keepdim=True).values.half().double()
    delta = ((x.max(-1, keepdim=True).values - low) / 15).half().double()
    steps = ((x - low) / delta).round().clamp(0, 15).nan_to_num(0.0)
    return (low + steps * delta).reshape(shape)


def _exact_cache(state, seq, head):
    """Keys and values [tokens, D] of one sequence's head, in 64 bits, read byte by byte from its pages."""
    case = state["case"]
    _, lengths, table = _views(state)
    tokens, groups = int(lengths[seq]), D // case["dims"]
    device = state["pages"].device
    t = torch.arange(tokens, device=device)
    place = table[seq].long()[t // case["page"]]
    tile_bytes = 16 * (D + 8 * groups)
    flat = state["pages"][0, :, head].reshape(-1)
    start = place * _page_bytes(case) + (t % case["page"]) // 16 * tile_bytes
    r = t % 16
    d = torch.arange(D, device=device)
    word, byte = d // 8, d % 8 // 2
    k_at = (word % 4 * 4 + word // 4) * 4 + byte
    v_at = d // 2 % 8 * 8 + d // 16

    def number(at):
        return (flat[(start + r * 64)[:, None] + at].long() // (1 + d % 2 * 15) % 16).double()

    def pair(which, part):
        at = (start + 2048 + r * 8 * groups)[:, None] + (which * groups + d // case["dims"]) * 4 + part * 2
        bits = flat[at].int() + flat[at + 1].int() * 256
        return bits.to(torch.int16).view(torch.float16).double()

    return number(k_at) * pair(0, 1) + pair(0, 0), number(1024 + v_at) * pair(1, 1) + pair(1, 0)


def _exact_attend(state):
    case = state["case"]
    group = case["q_heads"] // case["kv_heads"]
    q = state["queries"].double()
    out = torch.zeros_like(q)
    _, lengths, _ = _views(state)
    for b, seq in enumerate(state["seqs"].tolist()):
        tokens, count = int(lengths[seq]), int(state["counts"][b])
        if not tokens or not count:
            continue
        future = torch.arange(tokens, device=q.device) > (tokens - count + torch.arange(count, device=q.device))[:, None]
        for h in range(case["kv_heads"]):
            keys, values = _exact_cache(state, seq, h)
            part = slice(h * group, (h + 1) * group)
            logits = torch.einsum("ihd,td->hit", q[b, :count, part], keys) * D ** -0.5
            p = logits.masked_fill(future, -math.inf).softmax(-1)
            out[b, :count, part] = torch.einsum("hit,td->ihd", p, values)
    return out


def _exact_select(state):
    case = state["case"]
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros_like(state["queries"], dtype=torch.float64)
    for b, seq in enumerate(state["seqs"].tolist()):
        for h in range(case["kv_heads"]):
            keys, values = _exact_cache(state, seq, h)
            part = slice(h * group, (h + 1) * group)
            index = state["indices"][b, part]
            logits = torch.einsum("hd,hsd->hs", state["queries"][b, part].double(), keys[index]) * D ** -0.5
            if state["valid"] is not None:
                logits = logits.masked_fill(~state["valid"][b, part], -math.inf)
            p = logits.softmax(-1).nan_to_num(0.0)
            out[b, part] = torch.einsum("hs,hsd->hd", p, values[index])
    return out
