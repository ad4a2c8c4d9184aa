"""A host model of the 4-bit paged KV cache: bytes, tables and attention in plain loops.

Numbers and pairs follow the documented fp32 formula bit for bit; attention is in 64 bits.
"""
from __future__ import annotations

import numpy as np

D = 128


def quantise(x: np.ndarray, group: int):
    """Numbers 0..15 [..., 128] and fp16 low, delta [..., 128 / group] of float32 values."""
    x = np.where(np.isnan(x), np.float32(0), x.astype(np.float32))
    x = np.clip(x, np.float32(-65504), np.float32(65504)).reshape(*x.shape[:-1], D // group, group)
    low = x.min(-1).astype(np.float16)
    span = (x.max(-1) - low.astype(np.float32)) * (np.float32(1) / np.float32(15))
    delta = np.maximum(span, np.float32(0)).astype(np.float16)
    d32 = delta.astype(np.float32)
    scale = np.divide(np.float32(1), d32, out=np.zeros_like(d32), where=d32 > 0)
    n = np.rint((x - low.astype(np.float32)[..., None]) * scale[..., None])
    return np.clip(n, 0, 15).astype(np.uint8).reshape(*x.shape[:-2], D), low, delta


def values_of(n, low, delta, group):
    """float64 values that the numbers stand for."""
    return np.repeat(low.astype(np.float64), group, -1) + n * np.repeat(delta.astype(np.float64), group, -1)


class HostCache:
    """Tables and rows of the cache, as Python lists and arrays."""

    def __init__(self, num_pages, kv_heads, max_seqs, max_pages, page_size, group, layers=1):
        self.page_size, self.group, self.kv_heads = page_size, group, kv_heads
        self.refs = np.zeros(num_pages, np.int32)
        self.lengths = np.zeros(max_seqs, np.int32)
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        groups = D // group
        self.tile = 16 * (D + 8 * groups)
        self.pages = np.zeros((layers, num_pages, kv_heads, page_size // 16 * self.tile), np.uint8)

    @classmethod
    def like(cls, cache):
        """A host copy of a Kv4Cache."""
        host = cls(cache.num_pages, cache.kv_heads, cache.max_seqs, cache.max_pages, cache.page_size,
                   cache.dim_group_size, cache.layers)
        host.pull(cache)
        return host

    def pull(self, cache):
        self.refs = cache.refs.cpu().numpy().copy()
        self.lengths = cache.lengths.cpu().numpy().copy()
        self.table = cache.table.cpu().numpy().copy()
        self.pages = cache.pages.cpu().numpy().copy()

    def same_tables(self, cache):
        np.testing.assert_array_equal(self.refs, cache.refs.cpu().numpy(), err_msg="refs")
        np.testing.assert_array_equal(self.lengths, cache.lengths.cpu().numpy(), err_msg="lengths")
        np.testing.assert_array_equal(self.table, cache.table.cpu().numpy(), err_msg="table")

    def same(self, cache):
        self.same_tables(cache)
        np.testing.assert_array_equal(self.pages, cache.pages.cpu().numpy(), err_msg="pages")

    def held(self, tokens):
        return -(-tokens // self.page_size)

    # -- rows ---------------------------------------------------------------------
    def _row(self, layer, seq, head, position):
        """Views of one token's key bytes, value bytes and fp16 pairs [2, groups, 2]."""
        page = self.table[seq, position // self.page_size]
        at = position % self.page_size
        tile = self.pages[layer, page, head, at // 16 * self.tile:(at // 16 + 1) * self.tile]
        r, pairs = at % 16, 8 * (D // self.group)
        return (tile[r * 64:(r + 1) * 64], tile[1024 + r * 64:1024 + (r + 1) * 64],
                tile[2048 + r * pairs:2048 + (r + 1) * pairs])

    def put(self, layer, seq, head, position, key, value):
        kb, vb, pairs = self._row(layer, seq, head, position)
        (kn, kl, kd), (vn, vl, vd) = quantise(key, self.group), quantise(value, self.group)
        for w in range(16):
            for i in range(4):
                d = 8 * w + 2 * i
                kb[(w % 4 * 4 + w // 4) * 4 + i] = kn[d] | kn[d + 1] << 4
        for b in range(64):
            vb[b % 8 * 8 + b // 8] = vn[2 * b] | vn[2 * b + 1] << 4
        both = np.stack([np.stack([kl, kd], -1), np.stack([vl, vd], -1)])
        pairs[:] = both.reshape(-1).view(np.uint8)

    def get(self, layer, seq, head, position):
        """float64 key and value of a cached token."""
        kb, vb, pairs = self._row(layer, seq, head, position)
        kn, vn = np.zeros(D, np.uint8), np.zeros(D, np.uint8)
        for b in range(64):
            w, i = b // 4, b % 4
            byte = kb[(w % 4 * 4 + w // 4) * 4 + i]
            kn[2 * b], kn[2 * b + 1] = byte & 15, byte >> 4
            byte = vb[b % 8 * 8 + b // 8]
            vn[2 * b], vn[2 * b + 1] = byte & 15, byte >> 4
        p = pairs.copy().view(np.float16).reshape(2, D // self.group, 2)
        return (values_of(kn, p[0, :, 0], p[0, :, 1], self.group), values_of(vn, p[1, :, 0], p[1, :, 1], self.group))

    def rows(self, layer, seq, head, positions):
        got = [self.get(layer, seq, head, int(t)) for t in positions]
        if not got:
            return np.zeros((0, D)), np.zeros((0, D))
        return np.stack([k for k, _ in got]), np.stack([v for _, v in got])

    # -- pages --------------------------------------------------------------------
    def extend(self, seqs, counts):
        """False (and no change) when pages or columns are short."""
        plan, needed, seen = [], 0, set()
        for s, c in zip(seqs, counts):
            if not 0 <= s < len(self.lengths) or s in seen:
                continue
            seen.add(s)
            held, c = int(self.lengths[s]), max(0, c)
            copied = -1
            if c and held % self.page_size and self.refs[self.table[s, self.held(held) - 1]] > 1:
                copied = int(self.table[s, self.held(held) - 1])
            if self.held(held + c) > self.table.shape[1]:
                return False
            need = self.held(held + c) - self.held(held) + (copied >= 0)
            plan.append((s, c, copied, need))
            needed += need
        free = np.flatnonzero(self.refs == 0)
        if len(free) < needed:
            return False
        at = 0
        for s, c, copied, need in plan:
            held = int(self.lengths[s])
            column = self.held(held) - (copied >= 0)
            for j in range(need):
                self.table[s, column + j] = free[at + j]
                self.refs[free[at + j]] = 1
            if copied >= 0:
                self.refs[copied] -= 1
                self.pages[:, free[at]] = self.pages[:, copied]
            self.lengths[s] += c
            at += need
        return True

    def fork(self, parents, children):
        rows = [(self.table[p].copy(), self.lengths[p]) for p in parents]
        for (row, length), child in zip(rows, children):
            for page in row[:self.held(length)]:
                self.refs[page] += 1
        for (row, length), child in zip(rows, children):
            for page in self.table[child, :self.held(self.lengths[child])]:
                self.refs[page] -= 1
            self.table[child], self.lengths[child] = row, length

    def truncate(self, seqs, lengths):
        for s, length in zip(seqs, lengths):
            length = min(int(self.lengths[s]), max(0, int(length)))
            for j in range(self.held(length), self.held(int(self.lengths[s]))):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.lengths[s] = length

    def compact(self):
        live = int((self.refs > 0).sum())
        sources = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        targets = [p for p in range(live) if self.refs[p] == 0]
        place = dict(zip(sources, targets))
        for a, b in place.items():
            self.pages[:, b] = self.pages[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for at, page in np.ndenumerate(self.table):
            self.table[at] = place.get(int(page), page)
        return live, len(sources)


def attention(query: np.ndarray, keys: np.ndarray, values: np.ndarray, scale: float) -> np.ndarray:
    """One row over its tokens, float64; zeros when it sees none."""
    if not len(keys):
        return np.zeros(D)
    logits = keys @ query * scale
    p = np.exp(logits - logits.max())
    return p @ values / p.sum()


def verify(target, draft, tokens, count, uniforms, noise):
    """One sequence's tokens and accepted count; float32 arrays, comparisons and divisions in float32."""
    vocab, accepted = target.shape[1], 0
    while accepted < count:
        d = tokens[accepted]
        if not 0 <= d < vocab:
            break
        q = np.float32(1) if draft is None else draft[accepted, d]
        if not np.float32(uniforms[accepted] * q) < target[accepted, d]:
            break
        accepted += 1
    row = target[accepted]
    weight = row
    if accepted < count:
        over = row.copy()
        if draft is None:
            if 0 <= tokens[accepted] < vocab:
                over[tokens[accepted]] = 0
        else:
            over = np.maximum(row - draft[accepted], np.float32(0))
        weight = over if (over > 0).any() else row
    ratio = np.where(weight > 0, weight / noise, np.float32(-1))
    return list(tokens[:accepted]) + [int(np.argmax(ratio))] + [-1] * (len(tokens) - accepted), accepted
