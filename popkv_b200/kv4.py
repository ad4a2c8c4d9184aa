"""A KV cache held in 4 bits, in pages, and the attention that reads it.

``Kv4Cache`` holds keys and values of several sequences and layers as 4-bit numbers
with an fp16 (low, delta) pair per group of 32, 64 or 128 dims: 160, 144 or 136 bytes a
token and KV head instead of 512 in bf16.  Pages of 16 to 256 tokens are shared between
sequences (parallel samples, beams, drafted branches) and copied when a shared one is
written.  All tables live on the device; no call here synchronises except ``check`` and
``free_pages``.

A decode step, for the sequences ``seqs`` (int32 slots of the cache)::

    cache.extend(seqs, 1)                               # room for the token, in every layer
    for layer in ...:
        cache.write(keys, values, seqs=seqs, layer=layer)
        out = cache.attention(queries, seqs=seqs, layer=layer)              # dense layers
        out = cache.attention_selected(queries, indices, seqs=seqs, layer=layer)  # sparse layers

With drafted tokens, ``extend`` / ``write`` / ``attention`` take several tokens a sequence
(``counts`` when the drafts are of uneven length), ``popkv_b200.speculative.verify_drafts``
says how many stay, and ``truncate`` drops the rest.

The reference keeps a contiguous 16-bit cache of one sequence (popkv.py:965-972) and has no
counterpart.  The byte layout is documented in ``include/popkv_b200.h``.  Sequence ids of -1
are padding; ids out of range or repeated set an error bit that ``check`` raises on.  After an
``extend`` that found no room, ``extend`` and ``write`` do nothing until ``check`` has raised: the
cache stays as it was before that step, which can be repeated once pages are free.

Streams: calls run on the current stream of the cache's device.  Calls on one cache that
overlap in time must be ordered by the caller when one of them writes.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib

HEAD_DIM = 128
DIM_GROUP_SIZES = (32, 64, 128)
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQUENCES_PER_CALL = 4096


# Argument words of the calls that a decode step makes for each layer (see popkv_kv4_*_words).
_WRITE = struct.Struct("16q").pack
_READ = struct.Struct("10q").pack
_ATTENTION = struct.Struct("12qf4x4q").pack


class _Descriptor(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("pages", "refs", "lengths", "table", "status")] + [
        (name, ctypes.c_int64) for name in ("layers", "num_pages", "kv_heads", "page_size", "dim_group_size",
                                            "max_seqs", "max_pages")]


def page_bytes(page_size: int, dim_group_size: int) -> int:
    """Bytes of one page of one KV head."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if dim_group_size not in DIM_GROUP_SIZES:
        raise ValueError(f"dim_group_size must be one of {DIM_GROUP_SIZES}")
    return page_size * (HEAD_DIM + 8 * (HEAD_DIM // dim_group_size))


class Kv4Cache:
    """Pages, tables and operations of a 4-bit KV cache (head_dim 128).

    Args:
        num_pages: pages of the pool (of each layer).
        kv_heads, layers: KV heads and layers of the model.
        max_seqs: sequence slots.
        max_tokens: most tokens of one sequence (rounded up to whole pages).
        page_size: tokens of a page, one of 16, 32, 64, 128, 256.
        dim_group_size: dims that share a (low, delta) pair, one of 32, 64, 128.
    """

    def __init__(self, num_pages: int, *, kv_heads: int, layers: int = 1, max_seqs: int = 1, max_tokens: int,
                 page_size: int = 64, dim_group_size: int = 32, device="cuda") -> None:
        size = page_bytes(page_size, dim_group_size)
        if min(num_pages, kv_heads, layers, max_seqs, max_tokens) < 1:
            raise ValueError("cache sizes must be positive")
        max_pages = math.ceil(max_tokens / page_size)
        pages = torch.zeros((layers, num_pages, kv_heads, size), dtype=torch.uint8, device=device)
        tables = torch.zeros(num_pages + max_seqs * (1 + max_pages), dtype=torch.int32, device=device)
        tables[num_pages + max_seqs:] = -1
        self._bind(pages, tables, max_seqs, page_size, dim_group_size)

    @classmethod
    def from_tensors(cls, pages: torch.Tensor, tables: torch.Tensor, *, max_seqs: int, page_size: int,
                     dim_group_size: int) -> "Kv4Cache":
        """A cache over buffers that the caller holds.

        pages: uint8 [layers, num_pages, kv_heads, page_bytes]; tables: int32, refs [num_pages],
        lengths [max_seqs] and table [max_seqs, max_pages] one after another.  Both contiguous.
        """
        size = page_bytes(page_size, dim_group_size)
        if pages.ndim != 4 or pages.dtype != torch.uint8 or not pages.is_contiguous() or pages.shape[3] != size:
            raise ValueError(f"pages must be contiguous uint8 [layers, num_pages, kv_heads, {size}]")
        if min(pages.shape) < 1:
            raise ValueError("cache sizes must be positive")
        if tables.ndim != 1 or tables.dtype != torch.int32 or not tables.is_contiguous():
            raise ValueError("tables must be a contiguous int32 vector")
        if tables.device != pages.device:
            raise ValueError("pages and tables must share a device")
        rest = tables.numel() - int(pages.shape[1]) - max_seqs
        if max_seqs < 1 or rest < max_seqs or rest % max_seqs:
            raise ValueError("tables must hold refs [num_pages], lengths [max_seqs] and table [max_seqs, max_pages]")
        cache = cls.__new__(cls)
        cache._bind(pages, tables, max_seqs, page_size, dim_group_size)
        return cache

    def _bind(self, pages, tables, max_seqs, page_size, dim_group_size) -> None:
        self.pages, self.tables = pages, tables
        self.layers, self.num_pages, self.kv_heads = (int(x) for x in pages.shape[:3])
        self.max_seqs, self.page_size, self.dim_group_size = int(max_seqs), int(page_size), int(dim_group_size)
        self.refs = tables[:self.num_pages]
        self.lengths = tables[self.num_pages:self.num_pages + self.max_seqs]
        self.table = tables[self.num_pages + self.max_seqs:].view(self.max_seqs, -1)
        self.max_pages = int(self.table.shape[1])
        self.device = pages.device  # a CUDA device has its index here
        self.status = torch.zeros(4, dtype=torch.int32, device=pages.device)
        self._descriptor = _Descriptor(
            pages.data_ptr(), self.refs.data_ptr(), self.lengths.data_ptr(), self.table.data_ptr(),
            self.status.data_ptr(), self.layers, self.num_pages, self.kv_heads, self.page_size,
            self.dim_group_size, self.max_seqs, self.max_pages)
        self._address = ctypes.addressof(self._descriptor)
        self._workspaces = {}  # of each stream: the attention's scratch and the sizes it holds
        self._scratches = {}   # of each stream: the page operations' scratch

    # -- arguments -----------------------------------------------------------------
    def _call(self, entry, *args) -> None:
        index = self.device.index
        if index is None:
            raise RuntimeError("the 4-bit cache must be on a CUDA device")
        if torch.cuda.current_device() == index:
            status = entry(self._address, *args, _lib.raw_stream(index))
        else:
            with torch.cuda.device(index):
                status = entry(self._address, *args, _lib.raw_stream(index))
        if status:
            _lib.check(status)

    def _call_words(self, entry, pack, *args) -> None:
        index = self.device.index
        if index is None:
            raise RuntimeError("the 4-bit cache must be on a CUDA device")
        if torch.cuda.current_device() == index:
            status = entry(pack(self._address, *args, _lib.raw_stream(index)))
        else:
            with torch.cuda.device(index):
                status = entry(pack(self._address, *args, _lib.raw_stream(index)))
        if status:
            _lib.check(status)

    def _ids(self, ids, name: str) -> torch.Tensor:
        """int32 [n] on the cache's device, from a tensor or a sequence of ints."""
        if not isinstance(ids, torch.Tensor):
            ids = torch.tensor(ids, dtype=torch.int32, device=self.device)
        if ids.dtype is not torch.int32 or not ids.is_contiguous():
            if ids.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"{name} must be int32 or int64")
            # What does not fit becomes the nearest number that does: out of range, or longer than any sequence.
            ids = ids.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32).contiguous()
        if ids.ndim != 1:
            raise ValueError(f"{name} must be one-dimensional")
        if ids.device != self.device:
            raise RuntimeError(f"{name} must be on the cache's device")
        return ids

    def _sequences(self, seqs, name: str = "seqs", most: int = MAX_SEQUENCES_PER_CALL) -> tuple[torch.Tensor, int]:
        """The ids and their number."""
        seqs = self._ids(seqs, name)
        n = seqs.shape[0]
        if n > most:
            raise ValueError(f"at most {most} sequences in one call")
        return seqs, n

    def _per_sequence(self, values, n: int, name: str) -> torch.Tensor:
        values = self._ids(values, name)
        if values.shape[0] != n:
            raise ValueError(f"{name} must have one value per listed sequence")
        return values

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer must be in [0, {self.layers})")
        return layer

    def _scratch(self, numbers: int) -> torch.Tensor:
        """int32 scratch of a page operation, one buffer per stream (its own inside a graph capture)."""
        index = self.device.index
        if index is None or torch.cuda.is_current_stream_capturing():
            return torch.empty(numbers, dtype=torch.int32, device=self.device)
        key = _lib.raw_stream(index)
        held = self._scratches.get(key)
        if held is None or held.shape[0] < numbers:
            held = self._scratches[key] = torch.empty(numbers, dtype=torch.int32, device=self.device)
        return held

    # -- rows ----------------------------------------------------------------------
    def write(self, keys: torch.Tensor, values: torch.Tensor, *, seqs, layer: int = 0, counts=None) -> None:
        """Quantise the keys and values of the last tokens of each listed sequence.

        keys, values: fp32/fp16/bf16 [n, tokens, kv_heads, 128], or [n, kv_heads, 128] for one
        token; any strides with contiguous dims (slices of a fused projection).  They are the
        last ``tokens`` (or ``counts[i]`` <= tokens, the first of the row's) of sequence
        ``seqs[i]`` (each listed once), for which ``extend`` has made room.  After an ``extend`` that
        found none nothing is written until ``check`` has raised.
        """
        if keys.ndim == 3 and values.ndim == 3:
            keys, values = keys.unsqueeze(1), values.unsqueeze(1)
        seqs, n = self._sequences(seqs, most=1 << 30)
        shape = keys.shape
        if (len(shape) != 4 or shape != values.shape or shape[0] != n or shape[2] != self.kv_heads
                or shape[3] != HEAD_DIM):
            raise ValueError(f"keys and values must be [{n}, tokens, {self.kv_heads}, {HEAD_DIM}]")
        code = _lib.DTYPE_CODES.get(keys.dtype)
        if code is None or keys.dtype != values.dtype:
            raise RuntimeError("keys and values must share an fp32/fp16/bf16 dtype")
        if keys.device != self.device or values.device != self.device:
            raise RuntimeError("keys and values must be on the cache's device")
        k0, k1, k2, last = keys.stride()
        if last != 1:
            keys = keys.contiguous()
            k0, k1, k2, _ = keys.stride()
        v0, v1, v2, last = values.stride()
        if last != 1:
            values = values.contiguous()
            v0, v1, v2, _ = values.stride()
        counts = None if counts is None else self._per_sequence(counts, n, "counts")
        self._call_words(_lib.lib().popkv_kv4_write_words, _WRITE, self._layer(layer), seqs.data_ptr(), n,
                         0 if counts is None else counts.data_ptr(), keys.data_ptr(), values.data_ptr(), code,
                         shape[1], k0, k1, k2, v0, v1, v2)

    def read(self, seqs, *, start: int = 0, tokens: int, layer: int = 0,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """Cached tokens [start, start + tokens) as keys and values [n, tokens, kv_heads, 128].

        Rows past a sequence's end are zeros.
        """
        code = _lib.DTYPE_CODES.get(dtype)
        if code is None:
            raise RuntimeError("dtype must be fp32/fp16/bf16")
        if start < 0 or tokens < 0:
            raise ValueError("start and tokens must not be negative")
        seqs, n = self._sequences(seqs, most=1 << 30)
        keys, values = torch.empty((2, n, tokens, self.kv_heads, HEAD_DIM), dtype=dtype, device=self.device).unbind(0)
        self._call_words(_lib.lib().popkv_kv4_read_words, _READ, self._layer(layer), seqs.data_ptr(), n, start, tokens,
                         keys.data_ptr(), values.data_ptr(), code)
        return keys, values

    # -- attention -----------------------------------------------------------------
    def workspace(self, n: int, q_heads: int, q_len: int = 1) -> torch.Tensor:
        """Scratch for attention calls of up to these sizes, for the ``workspace`` arguments.

        Without one, calls keep one per stream; inside a graph capture each call would make and clear
        its own.  Calls that overlap in time need one each.
        """
        lib = _lib.lib()
        size = lib.popkv_kv4_attention_workspace(n, self.kv_heads, q_heads, q_len)
        if size < 0:
            raise ValueError("query heads must be a multiple of the cache's KV heads")
        made = torch.empty(size, dtype=torch.uint8, device=self.device)
        made[lib.popkv_kv4_attention_workspace(0, self.kv_heads, q_heads, q_len):].zero_()  # the counters
        return made

    def _workspace(self, given, n: int, q_heads: int, q_len: int) -> torch.Tensor:
        if given is not None:
            if given.dtype != torch.uint8 or not given.is_contiguous() or given.device != self.device:
                raise ValueError("workspace must be a tensor of workspace()")
            return given
        index = self.device.index
        if index is None or torch.cuda.is_current_stream_capturing():
            return self.workspace(n, q_heads, q_len)
        key = _lib.raw_stream(index)
        held = self._workspaces.get(key)
        if held is not None and held[1] >= n and held[2] >= q_heads and held[3] >= q_len:
            return held[0]
        sizes = (n, q_heads, q_len) if held is None else (max(n, held[1]), max(q_heads, held[2]), max(q_len, held[3]))
        made = self.workspace(*sizes)
        self._workspaces[key] = (made, *sizes)
        return made

    def _queries(self, queries: torch.Tensor, shape, n: int) -> tuple[torch.Tensor, tuple, int]:
        """Rows that start on 16 bytes, their strides and their type's code."""
        if shape[0] != n or shape[-1] != HEAD_DIM:
            raise ValueError(f"queries must be [{n}, ..., query heads, {HEAD_DIM}]")
        if shape[-2] < 1 or shape[-2] % self.kv_heads:
            raise ValueError("query heads must be a multiple of the cache's KV heads")
        dtype = queries.dtype
        if dtype != torch.bfloat16 and dtype != torch.float16:
            raise RuntimeError("queries must be fp16 or bf16")
        if queries.device != self.device:
            raise RuntimeError("queries must be on the cache's device")
        strides = queries.stride()
        if strides[-1] != 1 or queries.data_ptr() % 16 or strides[0] % 8 or strides[1] % 8 or strides[-2] % 8:
            # An axis with one entry may have any stride, which contiguous() leaves as it is and nothing follows.
            if strides[-1] != 1 or queries.data_ptr() % 16 or any(
                    s % 8 for s, size in zip(strides[:-1], shape) if size > 1):
                queries = queries.contiguous()
                if queries.data_ptr() % 16:
                    queries = queries.clone()
                strides = queries.stride()
        return queries, strides, _lib.DTYPE_CODES[dtype]

    def attention(self, queries: torch.Tensor, *, seqs, layer: int = 0, counts=None,
                  softmax_scale: float | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of each listed sequence's last tokens over all its tokens.

        queries: fp16/bf16 [n, q_len, q_heads, 128], or [n, q_heads, 128] for one token; row j of
        sequence i is its token ``lengths[seqs[i]] - counts[i] + j`` (``counts`` default q_len).
        Returns the same shape and type; rows past ``counts[i]``, and rows that see no token, are
        zeros.  ``softmax_scale`` defaults to 1 / sqrt(128).  The softmax is in fp32; its weights times a
        group's delta are rounded to fp16 for the product with the 4-bit numbers, which moves fp16 outputs
        from 2.1e-4 off 64 bits (their own rounding) to 2.9e-4, and bf16 ones from 1.6e-3 to 1.7e-3.
        """
        shape = queries.shape
        if len(shape) != 4 and len(shape) != 3:
            raise ValueError("queries must be [n, q_len, query heads, 128] or [n, query heads, 128]")
        seqs, n = self._sequences(seqs, most=65535)
        queries, strides, code = self._queries(queries, shape, n)
        if counts is not None:
            counts = self._per_sequence(counts, n, "counts")
        out = (torch.empty_like(queries) if queries.is_contiguous()
               else torch.empty(shape, dtype=queries.dtype, device=self.device))
        q_heads = shape[-2]
        q_len, token_stride = (shape[1], strides[1]) if len(shape) == 4 else (1, 0)
        scratch = self._workspace(workspace, n, q_heads, q_len)
        self._call_words(_lib.lib().popkv_kv4_attention_words, _ATTENTION, self._layer(layer), seqs.data_ptr(), n,
                         0 if counts is None else counts.data_ptr(), queries.data_ptr(), code, q_heads, q_len,
                         strides[0], token_stride, strides[-2], _scale(softmax_scale), scratch.data_ptr(),
                         scratch.shape[0], out.data_ptr())
        return out

    def attention_selected(self, queries: torch.Tensor, indices: torch.Tensor, *, seqs, layer: int = 0,
                           valid_mask: torch.Tensor | None = None, softmax_scale: float | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one token's query heads over the cached tokens that each selected.

        queries: fp16/bf16 [n, q_heads, 128]; indices: int64 [n, q_heads, selected] token positions
        (``popkv_cuda.topk``'s); valid_mask: bool of the same shape.  A slot that is masked, negative
        or past the sequence's end contributes nothing.  Returns [n, q_heads, 128].
        """
        shape, picked = queries.shape, indices.shape
        if len(shape) != 3:
            raise ValueError("queries must be [n, query heads, 128]")
        if len(picked) != 3 or picked[:2] != shape[:2]:
            raise ValueError("indices must be [n, query heads, selected tokens]")
        if indices.dtype != torch.int64:
            raise ValueError("indices must be int64")
        seqs, n = self._sequences(seqs, most=65535)
        queries, strides, code = self._queries(queries, shape, n)
        if indices.device != self.device:
            raise RuntimeError("indices and valid mask must be on the cache's device")
        indices = indices.contiguous()
        if valid_mask is not None:
            if valid_mask.shape != picked:
                raise ValueError("valid mask must match indices")
            if valid_mask.dtype != torch.bool and valid_mask.dtype != torch.uint8:
                raise ValueError("valid mask must be bool or uint8")
            if valid_mask.device != self.device:
                raise RuntimeError("indices and valid mask must be on the cache's device")
            valid_mask = valid_mask.contiguous()
        out = (torch.empty_like(queries) if queries.is_contiguous()
               else torch.empty(shape, dtype=queries.dtype, device=self.device))
        scratch = self._workspace(workspace, n, shape[1], 1)
        self._call_words(_lib.lib().popkv_kv4_attention_selected_words, _ATTENTION, self._layer(layer),
                         seqs.data_ptr(), n, queries.data_ptr(), code, shape[1], strides[0], strides[1],
                         indices.data_ptr(), picked[2], 0 if valid_mask is None else valid_mask.data_ptr(),
                         _scale(softmax_scale), scratch.data_ptr(), scratch.shape[0], out.data_ptr())
        return out

    # -- pages ---------------------------------------------------------------------
    def extend(self, seqs, tokens) -> None:
        """Room for ``tokens`` (an int, or int32 [n]) more tokens of each listed sequence.

        Takes the lowest free pages; a last page that is partly filled and shared with another
        sequence is copied first, in every layer (by every listed holder, even where all of them are
        listed).  All or nothing: without enough free pages nothing changes, further extends and
        writes do nothing either, and ``check`` raises.
        """
        seqs, n = self._sequences(seqs)
        counts, count = None, 0
        if isinstance(tokens, int):
            count = tokens
            if count < 0:
                raise ValueError("tokens must not be negative")
        else:
            counts = self._per_sequence(tokens, n, "tokens")
        workspace = self._scratch(self.num_pages + 3 * n)
        self._call(_lib.lib().popkv_kv4_extend, seqs.data_ptr(), n, None if counts is None else counts.data_ptr(),
                   count, workspace.data_ptr())

    def fork(self, parents, children) -> None:
        """Sequence ``children[i]`` becomes a copy of ``parents[i]`` that shares its pages.

        What a child held before is given back.  Every parent is read before any child changes,
        so one call can reorder beams (children distinct, parents repeated at will).
        """
        parents, n = self._sequences(parents, "parents")
        children, m = self._sequences(children, "children")
        if m != n:
            raise ValueError("parents and children must have the same length")
        workspace = self._scratch(n * (1 + self.max_pages))
        self._call(_lib.lib().popkv_kv4_fork, parents.data_ptr(), children.data_ptr(), n, workspace.data_ptr())

    def truncate(self, seqs, lengths) -> None:
        """Shorten each listed sequence to ``lengths[i]`` tokens (longer: unchanged)."""
        seqs, n = self._sequences(seqs)
        lengths = self._per_sequence(lengths, n, "lengths")
        self._call(_lib.lib().popkv_kv4_truncate, seqs.data_ptr(), n, lengths.data_ptr())

    def free(self, seqs) -> None:
        """Give back every page of the listed sequences."""
        seqs, n = self._sequences(seqs)
        self._call(_lib.lib().popkv_kv4_truncate, seqs.data_ptr(), n, None)

    def compact(self) -> None:
        """Move the live pages to the front of the pool (``status[1]`` then counts them).

        Live pages past the number of live pages move, in order, to the free pages below it, in
        order; the tables follow.  The tail of the pool is then free.
        """
        workspace = self._scratch(3 * self.num_pages)
        self._call(_lib.lib().popkv_kv4_compact, workspace.data_ptr())

    def copy_pages(self, sources, targets) -> None:
        """Copy page ``sources[i]`` to page ``targets[i]`` in every layer (no table changes)."""
        sources, targets = self._ids(sources, "sources"), self._ids(targets, "targets")
        if sources.shape != targets.shape:
            raise ValueError("sources and targets must have the same length")
        self._call(_lib.lib().popkv_kv4_copy_pages, sources.data_ptr(), targets.data_ptr(), sources.shape[0])

    # -- state ---------------------------------------------------------------------
    def check(self) -> None:
        """Raise if a page operation failed since the last check (synchronises)."""
        bits = int(self.status[0].item())
        if not bits:
            return
        self.status[0] = 0
        reasons = [text for bit, text in ((1, "too few free pages or table columns for an extend"),
                                          (2, "a sequence id was out of range or repeated"),
                                          (4, "an attention gave up waiting for its copies")) if bits & bit]
        raise RuntimeError("4-bit cache: " + "; ".join(reasons))

    def free_pages(self) -> int:
        """Free pages of the pool (synchronises)."""
        return int((self.refs == 0).sum().item())


def _scale(softmax_scale: float | None) -> float:
    return HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
