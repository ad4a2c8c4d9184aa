"""The 4-bit cache and drafted-token verification without a GPU: layout, host checks, the host model itself."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from popkv_b200 import _lib
from popkv_b200 import kv4
from popkv_b200.speculative import verify_drafts
from tests import kv4_reference as R


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().exists():
        from popkv_b200 import build
        build.build()
    return _lib.lib()


def descriptor(**changes):
    values = dict(pages=4096, refs=16, lengths=16, table=16, status=16, layers=2, num_pages=8, kv_heads=2,
                  page_size=64, dim_group_size=32, max_seqs=3, max_pages=4)
    values.update(changes)
    d = kv4._Descriptor(**values)
    return d, ctypes.addressof(d)


def refused(lib, status, text, code=1):
    assert status == code and text in lib.popkv_last_error().decode(), lib.popkv_last_error()


@pytest.mark.parametrize("changes,text", [
    ({"pages": None}, "null buffer"), ({"pages": 4104}, "16-byte aligned"), ({"status": None}, "null buffer"),
    ({"dim_group_size": 16}, "dim_group_size"), ({"page_size": 48}, "page_size"), ({"page_size": 512}, "page_size"),
    ({"layers": 0}, "sizes out of range"), ({"num_pages": 0}, "sizes out of range"),
    ({"max_pages": 1 << 28}, "sizes out of range"), ({"kv_heads": 1 << 20}, "sizes out of range"),
])
def test_every_entry_checks_the_cache(lib, changes, text):
    keep, c = descriptor(**changes)
    p = ctypes.c_void_p(64)
    refused(lib, lib.popkv_kv4_write(c, 0, p, 1, None, p, p, 2, 1, 1, 1, 1, 1, 1, 1, None), text)
    refused(lib, lib.popkv_kv4_read(c, 0, p, 1, 0, 1, p, p, 2, None), text)
    refused(lib, lib.popkv_kv4_extend(c, p, 1, None, 1, p, None), text)
    refused(lib, lib.popkv_kv4_fork(c, p, p, 1, p, None), text)
    refused(lib, lib.popkv_kv4_truncate(c, p, 1, None, None), text)
    refused(lib, lib.popkv_kv4_compact(c, p, None), text)
    refused(lib, lib.popkv_kv4_copy_pages(c, p, p, 1, None), text)
    refused(lib, lib.popkv_kv4_extend(None, p, 1, None, 1, p, None), "null cache")


def test_entries_check_their_arguments(lib):
    keep, c = descriptor()
    p = ctypes.c_void_p(64)
    refused(lib, lib.popkv_kv4_write(c, 2, p, 1, None, p, p, 2, 1, 1, 1, 1, 1, 1, 1, None), "layer out of range")
    refused(lib, lib.popkv_kv4_write(c, 0, p, 1, None, p, p, 5, 1, 1, 1, 1, 1, 1, 1, None), "fp32/fp16/bf16")
    refused(lib, lib.popkv_kv4_write(c, 0, p, -1, None, p, p, 2, 1, 1, 1, 1, 1, 1, 1, None), "sizes out of range")
    refused(lib, lib.popkv_kv4_write(c, 0, p, 1, None, None, p, 2, 1, 1, 1, 1, 1, 1, 1, None), "null pointer")
    refused(lib, lib.popkv_kv4_read(c, 0, p, 1, -1, 1, p, p, 2, None), "sizes out of range")
    refused(lib, lib.popkv_kv4_extend(c, p, 5000, None, 1, p, None), "4096 sequences")
    refused(lib, lib.popkv_kv4_extend(c, p, 1, None, -1, p, None), "count out of range")
    refused(lib, lib.popkv_kv4_extend(c, p, 1, None, 1, None, None), "null pointer")
    refused(lib, lib.popkv_kv4_fork(c, p, None, 1, p, None), "null pointer")
    refused(lib, lib.popkv_kv4_copy_pages(c, p, p, -1, None), "count out of range")
    refused(lib, lib.popkv_verify_drafts(p, 1, 1, p, 1, 1, 9, 1, 1, 10, p, None, p, p, p, p, p, None), "fp32/fp16/bf16")
    refused(lib, lib.popkv_verify_drafts(p, 1, 1, p, 1, 1, 0, 1, 1, 0, p, None, p, p, p, p, p, None), "sizes out of range")
    refused(lib, lib.popkv_verify_drafts(p, 1, 1, p, 1, 1, 0, 1, 2000, 10, p, None, p, p, p, p, p, None), "sizes out of")
    refused(lib, lib.popkv_verify_drafts(p, 1, 1, p, 1, 1, 0, 1, 1, 10, None, None, p, p, p, p, p, None), "null pointer")
    refused(lib, lib.popkv_verify_drafts(p, 1, 1, p, 1, 1, 0, 1, 1, 10, p, None, p, p, None, p, p, None), "workspace")
    refused(lib, lib.popkv_kv4_attention(c, 0, p, 1, None, p, 2, 3, 1, 8, 8, 8, 1.0, p, 1 << 30, p, None), "multiple of")
    refused(lib, lib.popkv_kv4_attention(c, 0, p, 1, None, p, 0, 4, 1, 8, 8, 8, 1.0, p, 1 << 30, p, None), "fp16 or bf16")
    refused(lib, lib.popkv_kv4_attention(c, 0, p, 1, None, p, 2, 4, 1, 8, 8, 4, 1.0, p, 1 << 30, p, None), "aligned")
    refused(lib, lib.popkv_kv4_attention(c, 0, p, 1, None, p, 2, 4, 1, 8, 8, 8, 1.0, p, 100, p, None), "workspace")
    refused(lib, lib.popkv_kv4_attention(c, 2, p, 1, None, p, 2, 4, 1, 8, 8, 8, 1.0, p, 100, p, None), "layer out of")
    refused(lib, lib.popkv_kv4_attention_selected(c, 0, p, 1, p, 2, 4, 8, 8, None, 5, None, 1.0, p, 1 << 30, p, None),
            "null pointer")
    refused(lib, lib.popkv_kv4_attention_selected(c, 0, p, 1, p, 2, 4, 8, 8, p, -1, None, 1.0, p, 1 << 30, p, None),
            "selected out of range")
    assert lib.popkv_kv4_attention_workspace(1, 2, 3, 1) == -1 and lib.popkv_kv4_attention_workspace(1, 2, 4, 1) > 0
    # Nothing to do is no error, and needs no GPU.
    assert lib.popkv_kv4_extend(c, None, 0, None, 1, None, None) == 0
    assert lib.popkv_kv4_write(c, 0, None, 0, None, None, None, 2, 1, 1, 1, 1, 1, 1, 1, None) == 0


def test_python_surface_without_a_gpu():
    assert kv4.page_bytes(64, 32) == 64 * 160 and kv4.page_bytes(16, 128) == 16 * 136
    with pytest.raises(ValueError, match="page_size"):
        kv4.page_bytes(48, 32)
    with pytest.raises(ValueError, match="dim_group_size"):
        kv4.Kv4Cache(4, kv_heads=1, max_tokens=10, dim_group_size=16, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        kv4.Kv4Cache(0, kv_heads=1, max_tokens=10, device="cpu")
    cache = kv4.Kv4Cache(4, kv_heads=2, layers=3, max_seqs=2, max_tokens=100, device="cpu")
    assert cache.pages.shape == (3, 4, 2, 64 * 160) and cache.max_pages == 2 and cache.free_pages() == 4
    assert cache.table.tolist() == [[-1, -1], [-1, -1]] and cache.lengths.tolist() == [0, 0]
    for call in (lambda: cache.extend([0], 1), lambda: cache.compact(), lambda: cache.read([0], tokens=1)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()
    again = kv4.Kv4Cache.from_tensors(cache.pages, cache.tables, max_seqs=2, page_size=64, dim_group_size=32)
    assert again.max_pages == 2 and again.table.data_ptr() == cache.table.data_ptr()
    for pages, tables, kwargs in ((cache.pages[..., :-1], cache.tables, {}), (cache.pages.int(), cache.tables, {}),
                                  (cache.pages, cache.tables.long(), {}), (cache.pages, cache.tables[:-1], {}),
                                  (cache.pages, cache.tables, {"max_seqs": 0})):
        with pytest.raises(ValueError):
            kv4.Kv4Cache.from_tensors(pages, tables, **{"max_seqs": 2, "page_size": 64, "dim_group_size": 32, **kwargs})
    with pytest.raises(RuntimeError, match="CUDA device"):
        verify_drafts(torch.rand(1, 2, 5), torch.zeros(1, 1, dtype=torch.int64), torch.rand(1, 1), torch.rand(1, 5))


def test_host_model_stores_and_reads_what_it_was_given():
    rng = np.random.default_rng(0)
    for group in (32, 64, 128):
        host = R.HostCache(3, 2, 1, 3, 32, group)
        assert host.extend([0], [40])
        x = rng.standard_normal((2, 40, 2, 128)).astype(np.float32)
        for t in range(40):
            for h in range(2):
                host.put(0, 0, h, t, x[0, t, h], x[1, t, h])
        for t in range(40):
            for h in range(2):
                for which, got in enumerate(host.get(0, 0, h, t)):
                    n, low, delta = R.quantise(x[which, t, h], group)
                    np.testing.assert_array_equal(got, R.values_of(n, low, delta, group))
                    # Half a step, the fp16 rounding of low, and 15 times that of delta.
                    step = np.repeat(delta.astype(np.float64), group)
                    slack = 2.0 ** -11 * (np.abs(x[which, t, h]).max() + 15 * step)
                    assert (np.abs(got - x[which, t, h]) <= step / 2 + 2 * slack).all()


def test_verification_model_keeps_the_target_distribution():
    """Summed over its random numbers, the model's first token has the target's probabilities."""
    rng = np.random.default_rng(1)
    p, q = np.float32([0.5, 0.2, 0.3, 0.0]), np.float32([0.1, 0.6, 0.2, 0.1])
    counts = np.zeros(4)
    n = 20000
    for _ in range(n):
        token = int(rng.choice(4, p=q.astype(np.float64) / q.astype(np.float64).sum()))
        out, _ = R.verify(np.stack([p, p]), q[None], [token], 1, rng.random(1, dtype=np.float32),
                          rng.standard_exponential(4).astype(np.float32))
        counts[out[0]] += 1
    want = p.astype(np.float64) * n
    assert (np.abs(counts - want) <= 5 * np.sqrt(want) + 1e-9).all()


def test_waits_that_steer_a_warp_are_voted_on():
    """A bounded wait ends lane by lane; a warp that goes on with shuffles and matrix products has to agree first."""
    for name in ("kv4_attention.cu", "gemv.cu"):
        text = (Path(kv4.__file__).parent / "csrc" / name).read_text()
        assert "mbar_wait(" in text
        assert not re.findall(r"(?:if|while)\s*\(\s*!?\s*mbar_wait\(|=\s*mbar_wait\(", text), name


@pytest.mark.parametrize("max_pages,page_size", [(1 << 58, 64), (1 << 60, 16), ((1 << 56) + 3, 256), ((1 << 24) + 1, 64)])
def test_table_widths_past_64_bits_are_refused(lib, max_pages, page_size):
    """Widths whose product with the page size wraps to a small number."""
    keep, c = descriptor(max_pages=max_pages, page_size=page_size)
    refused(lib, lib.popkv_kv4_truncate(c, None, 0, None, None), "sizes out of range")
    keep, c = descriptor(max_pages=1 << 24, page_size=64)
    assert lib.popkv_kv4_truncate(c, None, 0, None, None) == 0
