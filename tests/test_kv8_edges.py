"""Edges of the 8-bit paged cache's entry points, without a GPU."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest
from test_kv8 import INVALID, LIB, P, UNSUPPORTED, _append, _attention, _batch, _cache, _refused

torch = pytest.importorskip("torch")

from mogemma_b200.kv8 import KV8Batch, KV8Cache, set_debug  # noqa: E402


@pytest.mark.parametrize(("more", "ok"), [
    ({"table_stride": 100, "table_width": 2}, False),  # 2 pages of 32 hold 64 of the 96 positions
    ({"table_stride": 100, "table_width": 3}, True),
    ({"table_stride": 3, "table_width": 0}, True),
    ({"table_stride": 100, "table_width": -1}, False),
])
def test_max_ctx_is_held_to_the_tables_width(more, ok) -> None:
    """Of a table that is some columns of a wider one, the pitch says nothing about the ids that belong to a sequence."""
    n = ctypes.c_int64()
    if ok:  # past the batch's checks: refused for its heads
        _refused(LIB.mg_kv8_attention, _cache(), _batch(**more), _attention(num_heads=5), INVALID, "num_heads")
        return
    text = "table_width" if more["table_width"] < 0 else "page table"
    _refused(LIB.mg_kv8_append, _cache(), _batch(**more), _append(), INVALID, text)
    _refused(LIB.mg_kv8_attention, _cache(), _batch(**more), _attention(), INVALID, text)
    assert LIB.mg_kv8_attention_workspace(ctypes.byref(_cache()), ctypes.byref(_batch(**more)), 4,
                                          ctypes.byref(n)) == INVALID


@pytest.mark.parametrize("rows", [1, 4])
def test_a_column_slice_of_a_table_gives_its_own_width(rows) -> None:
    wide = torch.zeros(rows, 50, dtype=torch.int32)
    batch = KV8Batch.__new__(KV8Batch)  # its constructor wants CUDA tensors; the description reads no contents
    batch.q_start, batch.ctx_len = torch.zeros(rows + 1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    batch.err, batch.max_q, batch.max_ctx = torch.zeros(1, dtype=torch.int32), 4, 65
    batch.page_table = wide[:, 8:10]
    desc = batch._desc(7)
    assert desc.table_width == 2 and desc.table_stride == (50 if rows > 1 else 2)
    _refused(LIB.mg_kv8_append, _cache(), desc, _append(), INVALID, "page table")  # 65 positions, 2 pages of 32
    batch.page_table = wide[:, 8:11]
    _refused(LIB.mg_kv8_append, _cache(), batch._desc(7), _append(k_dev=P + 4), INVALID, "aligned")


def test_the_debug_hook_refuses_unknown_handoffs() -> None:
    for stall in (-2, 13, 1 << 20):
        with pytest.raises(ValueError, match="stall"):
            set_debug(0, stall)
    set_debug(5, 12)
    set_debug()


@pytest.mark.parametrize(("sizes", "text"), [
    ((0, 16, 1, 64), "num_pages"), ((4, 16, 0, 64), "kv_heads"), ((4, 16, 65536, 64), "kv_heads"),
    ((4, 8, 1, 64), "page_size"), ((4, 48, 1, 64), "page_size"), ((4, 512, 1, 64), "page_size"),
    ((4, 16, 1, 32), "head_dim"), ((4, 16, 1, 96), "head_dim"), ((4, 16, 1, 512), "head_dim")])
def test_a_cache_that_every_call_would_refuse_is_not_made(sizes, text) -> None:
    with pytest.raises(ValueError, match=text):
        KV8Cache(*sizes, device="cpu")  # its codes would be refused for that, but no memory is taken


@pytest.mark.parametrize("scale", [3.0e38, -3.0e38, 2.4e38])
def test_a_scale_whose_product_with_log2_e_overflows_is_refused(scale) -> None:
    """The kernels work in powers of two: an infinite factor would turn scores of zero into NaN."""
    _refused(LIB.mg_kv8_attention, _cache(), _batch(), _attention(scale=scale), INVALID, "finite scale")


def test_a_star_import_needs_no_torch() -> None:
    code = ("import sys; sys.modules['torch'] = None\nfrom mogemma_b200 import *\n"
            "assert SyncGemmaModel and AsyncGemmaModel and EmbeddingModel and GenerationConfig\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=False)
    assert run.returncode == 0, run.stderr
    from mogemma_b200 import KV8Batch as by_name

    assert by_name is KV8Batch


def test_more_single_tokens_than_a_grid_holds_are_refused() -> None:
    """2^20 sequences of 2^13 kv heads of 256 would be 2^31 CTAs, one beyond the largest grid."""
    cache = _cache(num_kv_heads=1 << 13, head_dim=256, token_stride=256, head_stride=8192, page_stride=1 << 26)
    batch = _batch(batch=1 << 20, max_q=1)
    _refused(LIB.mg_kv8_append, cache, batch, _append(num_heads=0), UNSUPPORTED, "too large")
