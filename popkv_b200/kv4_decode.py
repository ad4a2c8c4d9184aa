"""Sampling decode of a Llama-shaped model from a 4-bit paged KV cache.

``Kv4Decoder`` puts the 4-bit cache (``popkv_b200.kv4``) and drafted-token verification
(``popkv_b200.speculative``) to work as a serving loop does:

* a prompt is prefilled into one slot, ``fork`` shares its pages with further slots
  (parallel samples), and the first token that a branch writes copies only the last page;
* ``generate`` decodes all slots together, one token a step or, with a smaller draft model,
  several: the drafts of a step go through the target in one pass, ``verify_drafts`` keeps a
  prefix of them on the device, and ``truncate`` takes the rest out of both caches;
* with a ``RetrievalConfig`` the sparse layers attend over the PopKV selection (bit-plane
  scores, top-k) of each query head, read from the 4-bit cache;
* ``release`` frees slots and moves the pages that are left together.

The reference decodes one greedy token a call from a 16-bit cache of one sequence
(popkv.py:988-1115).  Projections are library GEMMs here; ``popkv_b200.decoder`` is the
graph-captured decode of one length of 16-bit caches.

``python -m popkv_b200.kv4_decode`` runs a small random model through all of it.
"""
from __future__ import annotations

from dataclasses import replace

import torch
import torch.nn.functional as F

from . import popkv, popkv_cuda
from .decoder import LlamaConfig, LlamaWeights, apply_rope, rms_norm, rope_tables
from .kv4 import Kv4Cache
from .speculative import verify_drafts


class Kv4Decoder:
    """Slots of sequences that one model decodes from a 4-bit cache.

    Args:
        weights: the model (bf16).
        max_seqs, max_tokens: slots, and most tokens of one (rounded up to whole pages).
        num_pages: pages of the pool; default enough for every slot at full length.
        retrieval: dense layers, budget and group sizes of the sparse layers' PopKV selection
            (single-token steps only); None: every layer attends over all tokens.
        seed: of the random numbers that sampling takes.
    """

    def __init__(self, weights: LlamaWeights, *, max_seqs: int, max_tokens: int, num_pages: int | None = None,
                 page_size: int = 64, dim_group_size: int = 32,
                 retrieval: popkv.RetrievalConfig | None = None, seed: int = 0) -> None:
        cfg = weights.config
        cfg.validate()
        if retrieval is not None:
            retrieval.validate()
        self.weights, self.cfg, self.retrieval = weights, cfg, retrieval
        self.device = weights.embed.device
        pages = -(-max_tokens // page_size) * max_seqs
        if pages == max_seqs:
            # Slots that share their only page all copy it before it is free: one page more for every two at most.
            # With more pages a slot, sharing the others saves at least as many.
            pages += max_seqs // 2
        self.cache = Kv4Cache(pages if num_pages is None else num_pages, kv_heads=cfg.num_key_value_heads,
                              layers=cfg.num_hidden_layers, max_seqs=max_seqs, max_tokens=max_tokens,
                              page_size=page_size, dim_group_size=dim_group_size, device=self.device)
        self.max_tokens = self.cache.max_pages * page_size  # every token that the cache has room for has its position
        self.cos, self.sin = rope_tables(cfg, self.max_tokens, self.device)
        self.generator = torch.Generator(device=self.device).manual_seed(seed)
        group = cfg.num_attention_heads // cfg.num_key_value_heads
        self.head_to_kv = torch.arange(cfg.num_attention_heads, device=self.device) // group
        self.sparse_layers = () if retrieval is None else tuple(
            l for l in range(cfg.num_hidden_layers) if l not in retrieval.full_layers)
        self.planes: dict[tuple[int, int], popkv.PopKVCache] = {}  # of each (slot, sparse layer)

    # -- model ---------------------------------------------------------------------
    def _project(self, layer, x: torch.Tensor, positions: torch.Tensor):
        """Rotated queries and keys and the values of x [..., T, H] at positions [..., T], heads last but one."""
        cfg = self.cfg
        qh, kh, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        qkv = F.linear(rms_norm(x, layer.input_norm, cfg.rms_norm_eps), layer.qkv).unflatten(-1, (qh + 2 * kh, d))
        cos, sin = self.cos[positions].unsqueeze(-2), self.sin[positions].unsqueeze(-2)
        q, k = apply_rope(qkv[..., :qh, :], cos, sin), apply_rope(qkv[..., qh:qh + kh, :], cos, sin)
        return q, k, qkv[..., qh + kh:, :]

    def _mlp(self, layer, hidden: torch.Tensor, attn: torch.Tensor) -> torch.Tensor:
        hidden = hidden + F.linear(attn.flatten(-2), layer.o)
        gate, up = F.linear(rms_norm(hidden, layer.post_norm, self.cfg.rms_norm_eps), layer.gate_up).chunk(2, -1)
        return hidden + F.linear(F.silu(gate) * up, layer.down)

    def _logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return F.linear(rms_norm(hidden, self.weights.norm, self.cfg.rms_norm_eps), self.weights.lm_head).float()

    @torch.inference_mode()
    def prefill(self, slot: int, ids: torch.Tensor) -> torch.Tensor:
        """Run a prompt [T] through the model into an empty slot; returns the last token's logits [V]."""
        tokens = int(ids.shape[0])
        seqs = [slot]
        for l in self.sparse_layers:
            self.planes.pop((slot, l), None)
        self.cache.free(seqs)
        self.cache.extend(seqs, tokens)
        self.cache.check()
        hidden = self.weights.embed[ids.to(self.device)]
        positions = torch.arange(tokens, device=self.device)
        group = self.cfg.num_attention_heads // self.cfg.num_key_value_heads
        for l, layer in enumerate(self.weights.layers):
            q, k, v = self._project(layer, hidden, positions)
            self.cache.write(k[None], v[None], seqs=seqs, layer=l)
            if l in self.sparse_layers:
                self.planes[slot, l] = popkv.build_popkv_cache(
                    k.transpose(0, 1).contiguous(), group_size=self.retrieval.group_size,
                    dim_group_size=self.retrieval.dim_group_size, reserve_tokens=self.max_tokens - tokens)
            heads = [t.transpose(0, 1)[None] for t in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1))]
            attn = F.scaled_dot_product_attention(*heads, is_causal=True)[0].transpose(0, 1)
            hidden = self._mlp(layer, hidden, attn)
        return self._logits(hidden[-1])

    @torch.inference_mode()
    def forward(self, slots: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """Append tokens [n, T] to the slots (int32 [n]); returns the logits [n, T, V] after each.

        With sparse layers T is 1.  Where there is no room it raises before anything is written, with
        every slot as it was (this synchronises).
        """
        n, count = tokens.shape
        if self.sparse_layers and count != 1:
            raise ValueError("the sparse layers take one token a step")
        listed = slots.tolist() if self.sparse_layers else []
        if any((s, l) not in self.planes for s in listed for l in self.sparse_layers):
            raise ValueError("a slot has no prompt")
        held = self._held(slots)
        positions = held.long()[:, None] + torch.arange(count, device=self.device)
        self.cache.extend(slots, count)
        try:
            self.cache.check()
        except RuntimeError:
            self._back_to(slots, held)
            raise
        hidden = self.weights.embed[tokens]
        for l, layer in enumerate(self.weights.layers):
            q, k, v = self._project(layer, hidden, positions.clamp_max(self.max_tokens - 1))
            self.cache.write(k, v, seqs=slots, layer=l)
            if l in self.sparse_layers:
                attn = torch.stack([self._selected(s, l, q[i, 0], k[i, 0]) for i, s in enumerate(listed)])[:, None]
            else:
                attn = self.cache.attention(q, seqs=slots, layer=l)
            hidden = self._mlp(layer, hidden, attn)
        return self._logits(hidden)

    def _held(self, slots: torch.Tensor) -> torch.Tensor:
        """Tokens of each slot (of an id that is none, whatever: the cache refuses it)."""
        return self.cache.lengths[slots.long().clamp(0, self.cache.max_seqs - 1)]

    def _back_to(self, slots: torch.Tensor, held: torch.Tensor) -> None:
        """Take the slots back to their first ``held`` tokens, after an error that has been raised."""
        self.cache.truncate(slots, held)
        self.cache.status[0] = 0  # ids that the error was about are among them once more

    def _selected(self, slot: int, layer: int, query: torch.Tensor, key: torch.Tensor) -> torch.Tensor:
        """A sparse layer's attention [QH, D] of a slot's newest token, which its planes do not hold yet."""
        planes = self.planes[slot, layer]
        prefix = planes.token_count
        scores = popkv_cuda.score(query[None].contiguous(), planes.packed, head_to_kv=self.head_to_kv, tokens=prefix,
                                  dim_group_size=planes.dim_group_size)
        indices = popkv.select_tokens(scores, budget=self.retrieval.budget, prefix_tokens=prefix)
        popkv.append_popkv(planes, key[:, None])
        return self.cache.attention_selected(query[None], indices, seqs=[slot], layer=layer)[0]

    # -- slots ---------------------------------------------------------------------
    def fork(self, parent: int, children: list[int]) -> None:
        """Branches of a slot: its pages are shared until one of them writes."""
        self.cache.fork([parent] * len(children), children)
        for child in children:
            for layer in self.sparse_layers:
                planes = self.planes[parent, layer]
                self.planes[child, layer] = replace(planes, packed=tuple(t.clone() for t in planes.packed))

    def release(self, slots: list[int]) -> None:
        """Free slots, and move the pages of the others to the front of the pool."""
        self.cache.free(slots)
        self.cache.compact()
        for key in [k for k in self.planes if k[0] in slots]:
            del self.planes[key]

    # -- decoding ------------------------------------------------------------------
    def _noise(self, n: int, generator: torch.Generator | None = None) -> torch.Tensor:
        return torch.empty((n, self.cfg.vocab_size), device=self.device).exponential_(
            generator=self.generator if generator is None else generator)

    def sample(self, logits: torch.Tensor, temperature: float = 1.0,
               generator: torch.Generator | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Tokens [n] drawn from logits [n, V], and the probabilities [n, V] that they were drawn from.

        generator: of the random numbers, instead of the decoder's own.
        """
        if not temperature > 0:
            raise ValueError("temperature must be positive")
        probs = (logits / temperature).softmax(-1)
        n = probs.shape[0]
        none = torch.empty((n, 0), device=self.device)
        tokens, _ = verify_drafts(probs[:, None], none.long(), none, self._noise(n, generator))
        return tokens[:, 0], probs

    @torch.inference_mode()
    def generate(self, slots: list[int], first: torch.Tensor, steps: int, *, draft: "Kv4Decoder | None" = None,
                 drafts: int = 4, temperature: float = 1.0) -> tuple[list[list[int]], float]:
        """Decode at least ``steps`` tokens in every slot, after the tokens ``first`` [n] that follow
        their prompts.  ``draft``: a model whose slots of the same numbers hold the same tokens, which
        proposes ``drafts`` tokens a step.  Returns each slot's tokens (``first`` included) and the
        tokens a slot gained per step.  A step without room raises and leaves both models' slots as the
        step before left them.
        """
        if draft is not None and (self.sparse_layers or draft.sparse_layers):
            raise ValueError("drafted tokens need dense attention: the sparse layers take one token a step")
        if not temperature > 0:
            raise ValueError("temperature must be positive")
        if draft is not None and drafts < 1:
            raise ValueError("drafts must be positive")
        if draft is not None and draft.cfg.vocab_size != self.cfg.vocab_size:
            raise ValueError("the draft model's vocabulary must be the target's")
        n = len(slots)
        seqs = torch.tensor(slots, dtype=torch.int32, device=self.device)
        pending = first.to(self.device)
        out = [[int(t)] for t in pending.tolist()]
        passes = 0
        while min(len(o) for o in out) < steps:
            passes += 1
            if draft is None:
                pending, _ = self.sample(self.forward(seqs, pending[:, None])[:, 0], temperature)
                kept = pending[:, None]
            else:
                base = self._held(seqs)
                proposed, proposals, token = [], [], pending
                try:
                    for _ in range(drafts):
                        # The target's random numbers: the draft's own may be the same as those that
                        # verify it (equal seeds), and the two have to be independent.
                        token, probs = draft.sample(draft.forward(seqs, token[:, None])[:, 0], temperature,
                                                    self.generator)
                        proposed.append(token)
                        proposals.append(probs)
                    draft.forward(seqs, token[:, None])  # the last draft's keys and values
                    proposed, proposals = torch.stack(proposed, 1), torch.stack(proposals, 1)
                    logits = self.forward(seqs, torch.cat([pending[:, None], proposed], 1))
                except RuntimeError:
                    draft._back_to(seqs, base)  # where the target's slots are
                    raise
                uniforms = torch.rand((n, drafts), device=self.device, generator=self.generator)
                kept, accepted = verify_drafts((logits / temperature).softmax(-1), proposed, uniforms, self._noise(n),
                                               draft_probs=proposals)
                pending = kept.gather(1, accepted.long()[:, None])[:, 0]
                for cache in (self.cache, draft.cache):
                    cache.truncate(seqs, base + 1 + accepted)
            for row, tokens in zip(out, kept.tolist()):
                row.extend(t for t in tokens if t >= 0)
        self.cache.check()
        if draft is not None:
            draft.cache.check()
        return out, (sum(len(o) for o in out) - n) / (n * max(1, passes))


def main() -> None:
    config = LlamaConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, intermediate_size=1024,
                         vocab_size=4096, num_hidden_layers=4)
    weights = LlamaWeights.random(config, std=0.05)
    small = LlamaWeights(replace(config, num_hidden_layers=2), weights.embed, weights.layers[:2], weights.norm,
                         weights.lm_head)
    target = Kv4Decoder(weights, max_seqs=5, max_tokens=1024)
    draft = Kv4Decoder(small, max_seqs=5, max_tokens=1024, seed=1)
    prompt = torch.randint(0, config.vocab_size, (400,), generator=torch.Generator().manual_seed(0))
    logits = target.prefill(0, prompt)
    draft.prefill(0, prompt)
    branches = [1, 2, 3, 4]
    for decoder in (target, draft):
        decoder.fork(0, branches)
    print(f"prompt of {len(prompt)} tokens in slot 0, shared by {branches}: "
          f"{target.cache.num_pages - target.cache.free_pages()} of {target.cache.num_pages} pages in use")
    first, _ = target.sample(logits.expand(4, -1))
    tokens, gain = target.generate(branches, first, 48, draft=draft, drafts=4)
    print(f"48 tokens in each branch, {gain:.2f} tokens a pass with 4 drafts; "
          f"{target.cache.num_pages - target.cache.free_pages()} pages in use")
    target.release([0, 2, 4])
    live, moved = target.cache.status[1:3].tolist()
    print(f"two branches kept: {live} pages at the front of the pool, {moved} of them moved")
    more, _ = target.generate([1, 3], torch.tensor([tokens[0][-1], tokens[2][-1]]), 16)
    print(f"16 more tokens a branch, one a pass: {[len(m) for m in more]}")


if __name__ == "__main__":
    main()
