"""Edges of mg_kv8_append and mg_kv8_attention on the GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from mogemma_b200.kv8 import KV8Batch  # noqa: E402
from test_gpu_kv8 import BF16, F16, F32, World, _check_append, _check_attention, _ints, _snapshot  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 30])
def test_a_column_slice_of_a_page_table(n) -> None:
    """Its own columns only: a bound beyond them is refused, and a context beyond them reported."""
    w = World([(n, 100), (n, 60), (n, 77)], kv_heads=1, dim=64, page=16)
    q = w.rand(w.rows, 2, 64, dtype=F16)
    want = w.cache.attention(w.batch, q)
    wide = torch.zeros(3, 40, dtype=torch.int32, device="cuda")
    wide[:, 20:27] = w.batch.page_table[:, :7]
    lens = w.batch.q_start, w.batch.ctx_len
    batch = KV8Batch(*lens, wide[:, 20:27], max_q=n, max_ctx=112)
    assert torch.equal(w.cache.attention(batch, q), want)
    batch.check()
    for max_ctx in (113, 640):
        beyond = KV8Batch(*lens, wide[:, 20:27], max_q=n, max_ctx=max_ctx)
        k = w.rand(w.rows, 1, 64)
        for call in (lambda: w.cache.attention(beyond, q), lambda: w.cache.append(beyond, k, k.clone())):
            with pytest.raises(ValueError, match="page table"):
                call()
    w.batch.ctx_len[1] = 113
    out = w.cache.attention(batch, q)
    with pytest.raises(RuntimeError, match="lengths"):
        batch.check()
    assert bool((out[n:2 * n] == 0).all()) and torch.equal(out[:n], want[:n])
