"""The 8-bit paged cache's entry points without a GPU: struct layouts, refused arguments, refused tensors."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

from mogemma_b200 import _core

HEADER = Path(__file__).resolve().parent.parent / "include" / "mogemma_b200.h"
LIB = _core.lib()
P = 0x10000  # an aligned address that is never read: every call here is refused before its launch


def _cache(**more):
    d = {"struct_size": ctypes.sizeof(_core.KV8CacheDesc), "num_pages": 8, "page_size": 32, "num_kv_heads": 2,
         "head_dim": 64, "k_dev": P, "v_dev": P, "k_scale_dev": P, "v_scale_dev": P, "page_stride": 4096,
         "head_stride": 2048, "token_stride": 64}
    return _core.KV8CacheDesc(**{**d, **more})


def _batch(**more):
    d = {"struct_size": ctypes.sizeof(_core.KV8BatchDesc), "batch": 3, "total_q": 7, "max_q": 4, "max_ctx": 96,
         "q_start_dev": P, "ctx_len_dev": P, "page_table_dev": P, "table_stride": 3, "err_dev": P}
    return _core.KV8BatchDesc(**{**d, **more})


def _append(**more):
    d = {"struct_size": ctypes.sizeof(_core.KV8AppendArgs), "dtype": _core.MG_BF16, "out_dtype": _core.MG_BF16,
         "num_heads": 4, "rope_len": 96, "q_dev": P, "k_dev": P, "v_dev": P, "q_out_dev": P, "cos_dev": P,
         "sin_dev": P}
    d.update({n: 64 for n, _ in _core.KV8AppendArgs._fields_ if n.endswith("_stride")})
    return _core.KV8AppendArgs(**{**d, **more})


def _attention(**more):
    d = {"struct_size": ctypes.sizeof(_core.KV8AttentionArgs), "dtype": _core.MG_F16, "num_heads": 4, "scale": 0.1,
         "q_dev": P, "out_dev": P, "workspace_dev": P, "workspace_bytes": 1 << 40}
    d.update({n: 64 for n, _ in _core.KV8AttentionArgs._fields_ if n.endswith("_stride")})
    return _core.KV8AttentionArgs(**{**d, **more})


def _refused(fn, cache, batch, args, status, text) -> None:
    assert fn(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(args), None) == status
    assert text in LIB.mg_last_error().decode()


INVALID, UNSUPPORTED = _core.MG_ERR_INVALID, 6


@pytest.mark.parametrize(("more", "status", "text"), [
    ({"struct_size": 8}, INVALID, "struct_size"),
    ({"head_dim": 80}, UNSUPPORTED, "head_dim"),
    ({"head_dim": 512}, UNSUPPORTED, "head_dim"),
    ({"page_size": 8}, UNSUPPORTED, "page_size"),
    ({"page_size": 48}, UNSUPPORTED, "page_size"),
    ({"page_size": 512}, UNSUPPORTED, "page_size"),
    ({"num_pages": 0}, INVALID, "num_pages"),
    ({"num_kv_heads": 0}, INVALID, "num_kv_heads"),
    ({"k_dev": None}, INVALID, "null cache"),
    ({"v_scale_dev": None}, INVALID, "null cache"),
    ({"v_dev": P + 8}, INVALID, "16 bytes"),
    ({"token_stride": 72}, INVALID, "16 bytes"),
    ({"head_stride": 2050}, INVALID, "16 bytes"),
    ({"token_stride": 48}, INVALID, "at least head_dim"),
])
def test_bad_caches_are_refused(more, status, text) -> None:
    _refused(LIB.mg_kv8_append, _cache(**more), _batch(), _append(), status, "mg_kv8_append: ")
    _refused(LIB.mg_kv8_append, _cache(**more), _batch(), _append(), status, text)
    _refused(LIB.mg_kv8_attention, _cache(**more), _batch(), _attention(), status, text)


@pytest.mark.parametrize(("more", "status", "text"), [
    ({"struct_size": 0}, INVALID, "struct_size"),
    ({"batch": 0}, INVALID, "batch"),
    ({"total_q": 0}, INVALID, "total_q"),
    ({"max_q": -1}, INVALID, "max_q"),
    ({"max_ctx": 0}, INVALID, "max_ctx"),
    ({"table_stride": 0}, INVALID, "table_stride"),
    ({"max_ctx": 97}, INVALID, "page table"),
    ({"batch": 1 << 24}, UNSUPPORTED, "too large"),
    ({"q_start_dev": None}, INVALID, "null batch"),
    ({"err_dev": None}, INVALID, "null batch"),
])
def test_bad_batches_are_refused(more, status, text) -> None:
    _refused(LIB.mg_kv8_append, _cache(), _batch(**more), _append(), status, text)
    _refused(LIB.mg_kv8_attention, _cache(), _batch(**more), _attention(), status, text)


@pytest.mark.parametrize(("more", "status", "text"), [
    ({"struct_size": 1}, INVALID, "struct_size"),
    ({"dtype": _core.MG_U8}, UNSUPPORTED, "dtype"),
    ({"out_dtype": _core.MG_F16}, UNSUPPORTED, "out_dtype"),
    ({"k_dev": None}, INVALID, "null k or v"),
    ({"q_out_dev": None}, INVALID, "null q or q_out"),
    ({"num_heads": 3}, INVALID, "multiple of num_kv_heads"),
    ({"num_heads": -2}, INVALID, "multiple of num_kv_heads"),
    ({"sin_dev": None}, INVALID, "cos and sin"),
    ({"rope_len": 95}, INVALID, "rope_len"),
    ({"k_dev": P + 4}, INVALID, "aligned"),
    ({"dtype": _core.MG_F32, "k_dev": P + 8}, INVALID, "aligned"),
    ({"out_row_stride": 66}, INVALID, "multiples of 4"),
    ({"cos_dev": P + 4}, INVALID, "16 bytes"),
])
def test_bad_appends_are_refused(more, status, text) -> None:
    _refused(LIB.mg_kv8_append, _cache(), _batch(), _append(**more), status, text)


@pytest.mark.parametrize(("more", "status", "text"), [
    ({"struct_size": 1}, INVALID, "struct_size"),
    ({"dtype": _core.MG_F32}, UNSUPPORTED, "dtype"),
    ({"num_heads": 0}, INVALID, "num_heads"),
    ({"num_heads": 5}, INVALID, "num_heads"),
    ({"num_heads": 258}, UNSUPPORTED, "128 heads"),
    ({"window": -1}, INVALID, "window"),
    ({"scale": float("nan")}, INVALID, "finite scale"),
    ({"scale": float("inf")}, INVALID, "finite scale"),
    ({"q_dev": None}, INVALID, "null q or out"),
    ({"out_dev": P + 8}, INVALID, "16-byte aligned"),
    ({"q_head_stride": 68}, INVALID, "multiples of 8"),
])
def test_bad_attentions_are_refused(more, status, text) -> None:
    _refused(LIB.mg_kv8_attention, _cache(), _batch(), _attention(**more), status, text)


def test_answers_over_the_queries_are_refused() -> None:
    """Attention answers a row while other CTAs may still read it; the append may, but only element for element."""
    _refused(LIB.mg_kv8_attention, _cache(), _batch(), _attention(), INVALID, "out must not be q")
    text = "q_out may be q only"
    _refused(LIB.mg_kv8_append, _cache(), _batch(), _append(out_row_stride=128), INVALID, text)
    _refused(LIB.mg_kv8_append, _cache(), _batch(), _append(dtype=_core.MG_F32), INVALID, text)


def test_null_arguments_are_refused() -> None:
    c, b = ctypes.byref(_cache()), ctypes.byref(_batch())
    assert LIB.mg_kv8_append(None, b, ctypes.byref(_append()), None) == INVALID
    assert LIB.mg_kv8_append(c, None, ctypes.byref(_append()), None) == INVALID
    assert LIB.mg_kv8_append(c, b, None, None) == INVALID
    assert LIB.mg_kv8_attention(c, b, None, None) == INVALID
    assert LIB.mg_kv8_attention_workspace(c, b, 4, None) == INVALID


def test_struct_layouts_match_the_header(tmp_path: Path) -> None:
    names = {"mg_kv8_cache": _core.KV8CacheDesc, "mg_kv8_batch": _core.KV8BatchDesc,
             "mg_kv8_append_args": _core.KV8AppendArgs, "mg_kv8_attention_args": _core.KV8AttentionArgs}
    lines = [f'printf("%zu\\n", offsetof({c}, {f}));' for c, s in names.items() for f, _ in s._fields_]
    lines += [f'printf("%zu\\n", sizeof({c}));' for c in names]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mogemma_b200.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    try:
        subprocess.run(["gcc", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    except FileNotFoundError:
        pytest.skip("no C compiler")
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(s, f).offset for s in names.values() for f, _ in s._fields_]
    assert got == want + [ctypes.sizeof(s) for s in names.values()]


def test_tensors_off_the_gpu_are_refused() -> None:
    torch = pytest.importorskip("torch")
    from mogemma_b200 import KV8Batch, KV8Cache

    codes = torch.zeros(2, 1, 16, 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        KV8Cache.wrap(codes, codes, torch.ones(2, 1, 1), torch.ones(2, 1, 1))
    with pytest.raises(ValueError, match="page_size"):
        KV8Cache(2, 24, 1, 64)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        KV8Batch(ints, ints[:1], ints[None], max_q=1, max_ctx=16)
