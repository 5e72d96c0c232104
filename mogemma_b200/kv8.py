"""The 8-bit paged key/value cache on torch tensors: ``mg_kv8_append`` and ``mg_kv8_attention``.

``KV8Cache`` holds one layer's pages, ``KV8Batch`` the sequences of a step.
``append`` stores a step's new keys and values (head norm and rotation on the
way) and rotates its queries; ``attention`` answers them.  The definitions,
bounds and error rules are those of ``include/mogemma_b200.h``.

    cache = KV8Cache(num_pages=512, page_size=64, kv_heads=4, head_dim=256)
    batch = KV8Batch(q_start, ctx_len, page_table, max_q=1, max_ctx=8192)
    cache.append(batch, k, v, q=q, q_out=q, cos=cos, sin=sin, q_norm=wq, k_norm=wk)
    cache.attention(batch, q, out, scale=256 ** -0.5)

``append_call`` / ``attention_call`` check and bind the same arguments once; the
object they return launches the call each time it is called (on torch's current
stream of the cache's device; the caller orders its own tensors between streams,
the call its workspace and error word), so a decode loop that keeps its buffers pays for
the checks once.  A bound call reads the tensors' contents anew every time: new
rows, lengths and tables are written into the same tensors.  It may be captured
into a CUDA graph; the call object then has to live as long as the graph.

An attention call has a workspace of its own unless one is given: up to 39 MB
(prompts).  Calls that may run at the same time must not share
one; calls that follow each other may, as a model's layers should:

    ws = torch.empty(cache.workspace_bytes(batch, heads), dtype=torch.uint8, device="cuda")
    calls = [c.attention_call(batch, q, out, workspace=ws) for c in caches]
"""

from __future__ import annotations

import ctypes
from collections.abc import Callable
from typing import Any

import torch

from . import _core

BLOCK = 16  # tokens per scale (MG_KV8_BLOCK)
# MG_KV8_ERR_*
_ERRORS = {0x70000: "lengths out of bounds", 0x80000: "page id out of range",
           0x90000: "a device wait ran out; the answers are not complete"}
_TYPES = {torch.float32: _core.MG_F32, torch.bfloat16: _core.MG_BF16, torch.float16: _core.MG_F16}


# The current stream's handle without making a torch.cuda.Stream of it (3 us a call).
_raw_stream: Callable[[int], int] = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (  # noqa: SLF001
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _i32(x: int) -> int:
    """An int32 field's value; what it cannot hold becomes its nearest end, not the low bits."""
    return min(max(int(x), -(2**31)), 2**31 - 1)


def _rows(name: str, x: torch.Tensor, device: torch.device, dim: int) -> torch.Tensor:
    _need(isinstance(x, torch.Tensor) and x.dim() == 3 and x.shape[2] == dim and x.stride(2) == 1,
          f"{name} must be a [rows, heads, {dim}] tensor, contiguous along its last dimension")
    _need(x.device == device, f"{name} is on {x.device}, the cache on {device}")
    _need(x.dtype in _TYPES, f"{name} must be float32, bfloat16 or float16")
    return x


def _strides(x: torch.Tensor) -> tuple[int, int]:
    """Row and head strides; a dimension of size 1 may report any, and uses none."""
    return (x.stride(0) if x.shape[0] > 1 else 0), (x.stride(1) if x.shape[1] > 1 else 0)


def _written(name: str, x: torch.Tensor) -> None:
    # one stride spans a vector and the other all of the smaller dimension: rows and heads do not overlap
    (r, h), (nr, nh, d) = _strides(x), x.shape
    apart = (nr == 1 or r >= d) and (nh == 1 or h >= d)
    apart = apart and (nr == 1 or nh == 1 or r >= h * nh or h >= r * nr)
    _need(apart, f"{name} is written: its rows and heads must not overlap")


def _vector(name: str, x: torch.Tensor | None, device: torch.device, shape: tuple[int, ...]) -> int | None:
    if x is None:
        return None
    _need(x.dtype == torch.float32 and x.device == device and x.is_contiguous() and tuple(x.shape) == shape,
          f"{name} must be a contiguous float32 tensor of shape {shape} on {device}")
    return x.data_ptr()


def set_debug(wait_budget_ns: int = 0, stall: int = -1) -> None:
    """Failure-detection test hook (``mg_kv8_set_debug``): budget of the waits inside this thread's later attention calls,
    and a hand-off that one CTA withholds."""
    _core._check(_core.lib().mg_kv8_set_debug(int(wait_budget_ns), int(stall)))  # noqa: SLF001


class KV8Call:
    """A checked call with its tensors; launches on torch's current stream each time it is called."""

    def __init__(self, fn: Callable[..., int], batch: KV8Batch, structs: tuple[Any, ...], keep: tuple[Any, ...],
                 own: tuple[torch.Tensor, ...] = ()) -> None:
        self._fn = fn
        self._device = batch.device
        self._structs = structs
        self._refs = tuple(ctypes.byref(s) for s in structs)
        self._keep = (batch, *keep)
        self._own = (batch.err, *own)  # the tensors that the caller does not see
        self._homes = {batch.stream, _raw_stream(self._device.index)}  # streams they were made on
        self._met = set(self._homes) if len(self._homes) == 1 else set()

    def _meet(self, stream: int) -> None:
        """On another stream: behind what made the call's own tensors, which then live until this stream is done."""
        if torch.cuda.is_current_stream_capturing():  # a capture begins with a wait for the device; the graph's owner keeps the call
            return
        here = torch.cuda.current_stream()
        for home in self._homes - {stream}:
            here.wait_stream(torch.cuda.ExternalStream(home) if home else torch.cuda.default_stream())
        for x in self._own:
            x.record_stream(here)
        self._met.add(stream)

    def __call__(self) -> None:
        dev = self._device.index
        if torch.cuda.current_device() != dev:
            with torch.cuda.device(dev):
                return self()
        stream = _raw_stream(dev)
        if stream not in self._met:
            self._meet(stream)
        status = self._fn(*self._refs, stream)
        if status:
            _core._check(status)  # noqa: SLF001
        return None


class KV8Batch:
    """The sequences of a step: packed new tokens, contexts and page lists (``mg_kv8_batch``).

    ``q_start`` [batch + 1], ``ctx_len`` [batch] and ``page_table`` [batch, pages] are int32 tensors on
    the cache's device; ``max_q`` and ``max_ctx`` bound the lengths they will ever hold."""

    def __init__(self, q_start: torch.Tensor, ctx_len: torch.Tensor, page_table: torch.Tensor, *, max_q: int,
                 max_ctx: int) -> None:
        for name, x, dims in (("q_start", q_start, 1), ("ctx_len", ctx_len, 1), ("page_table", page_table, 2)):
            _need(isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.dim() == dims and x.is_cuda,
                  f"{name} must be a {dims}-dimensional int32 tensor on a CUDA device")
            _need(x.device == q_start.device, "q_start, ctx_len and page_table must be on one device")
            _need(x.numel() > 0 and x.stride(-1) == 1, f"{name} must be contiguous and not empty")
        n = ctx_len.shape[0]
        _need(q_start.shape[0] == n + 1 and page_table.shape[0] == n,
              "q_start has batch + 1 entries, page_table one row per sequence")
        self.q_start, self.ctx_len, self.page_table = q_start, ctx_len, page_table
        self.max_q, self.max_ctx = _i32(max_q), _i32(max_ctx)
        self.device = q_start.device
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.stream = _raw_stream(self.device.index)  # that the error word was made on

    def check(self) -> None:
        """Raises if a call since the last check met lengths or page ids out of bounds.  Waits for the whole device: the
        calls may have gone to any of its streams."""
        torch.cuda.synchronize(self.device)
        code = int(self.err.item())
        if code:
            self.err.zero_()
            torch.cuda.synchronize(self.device)  # before a later call on another stream
            raise RuntimeError(f"8-bit cache: {_ERRORS.get(code, f'error word 0x{code:x}')}")

    def _desc(self, total_q: int) -> _core.KV8BatchDesc:
        # the table may be some columns of a wider one; a single row may report any stride
        n, width = self.page_table.shape
        return _core.KV8BatchDesc(
            ctypes.sizeof(_core.KV8BatchDesc), n, _i32(total_q), self.max_q, self.max_ctx, _i32(width),
            self.q_start.data_ptr(), self.ctx_len.data_ptr(), self.page_table.data_ptr(),
            width if n == 1 else self.page_table.stride(0), self.err.data_ptr())


def _check_sizes(pages: int, heads: int, size: int, dim: int) -> None:
    """What mg_kv8_append and mg_kv8_attention take: a cache of other sizes would be refused by every call."""
    _need(pages > 0 and 0 < heads <= 65535, "need num_pages > 0 and kv_heads in 1..65535")
    _need(size in (16, 32, 64, 128, 256), "page_size must be a power of two in 16..256")
    _need(dim in (64, 128, 256), "head_dim must be 64, 128 or 256")


class KV8Cache:
    """One layer's pages of e4m3 codes ``[pages, kv heads, page size, head dim]`` and their scales
    ``[pages, kv heads, page size / 16]``."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 device: torch.device | str = "cuda") -> None:
        _check_sizes(num_pages, kv_heads, page_size, head_dim)
        shape = (num_pages, kv_heads, page_size, head_dim)
        scales = (num_pages, kv_heads, page_size // BLOCK)
        self._bind(*(torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)),
                   *(torch.ones(scales, dtype=torch.float32, device=device) for _ in range(2)))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> KV8Cache:
        """A cache over existing tensors (float8_e4m3fn or uint8 codes; k and v with equal strides)."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        for x in (k, v):
            _need(isinstance(x, torch.Tensor) and x.dim() == 4 and x.is_cuda
                  and x.dtype in (torch.float8_e4m3fn, torch.uint8) and x.stride(3) == 1,
                  "codes must be 4-dimensional float8_e4m3fn or uint8 CUDA tensors, contiguous along the head dim")
        _need(k.shape == v.shape and k.stride() == v.stride() and k.device == v.device,
              "k and v must have the same shape, strides and device")
        pages, heads, size, dim = k.shape
        _check_sizes(pages, heads, size, dim)
        reach = 1  # bytes that the dimensions of smaller strides span
        for stride, n in sorted((s, n) for s, n in zip(k.stride(), k.shape) if n > 1):
            _need(stride >= reach, "pages, heads and tokens of the cache must not overlap")
            reach += stride * (n - 1)
        _need(k.data_ptr() != v.data_ptr() and k_scale.data_ptr() != v_scale.data_ptr(),
              "k and v must not be the same memory, nor their scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self.device = k.device
        shape = (pages, heads, size // BLOCK)
        ks, vs = (_vector(n, x, self.device, shape) for n, x in (("k_scale", k_scale), ("v_scale", v_scale)))
        # strides of dimensions of size 1 say nothing: give the dense ones
        token = k.stride(2)
        head = k.stride(1) if heads > 1 else max(token * size, dim)
        page = k.stride(0) if pages > 1 else max(head * heads, dim)
        self._c = _core.KV8CacheDesc(ctypes.sizeof(_core.KV8CacheDesc), pages, size, heads, dim, 0, k.data_ptr(),
                                     v.data_ptr(), ks, vs, page, head, token)

    def _batch(self, batch: KV8Batch, total_q: int) -> _core.KV8BatchDesc:
        _need(batch.device == self.device, f"the batch is on {batch.device}, the cache on {self.device}")
        return batch._desc(total_q)  # noqa: SLF001

    # ------------------------------------------------------------------ append
    def append_call(self, batch: KV8Batch, k: torch.Tensor, v: torch.Tensor, *, q: torch.Tensor | None = None,
                    q_out: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                    k_norm: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                    sin: torch.Tensor | None = None) -> KV8Call:
        """Binds ``mg_kv8_append``: k, v [rows, kv heads, head dim] and, with its rotated copy q_out (or q itself),
        q [rows, heads, head dim]; norm weights [head dim]; cos / sin [positions, head dim / 2]."""
        d = self.head_dim
        for name, x in (("k", k), ("v", v)):
            _rows(name, x, self.device, d)
            _need(x.shape[1] == self.kv_heads and x.dtype == k.dtype and x.shape[0] == k.shape[0],
                  f"{name} must have {self.kv_heads} heads, and k and v the same rows and type")
        _need((q is None) == (q_out is None), "q and q_out come together")
        heads, out_dtype = 0, k.dtype
        if q is not None:
            _rows("q", q, self.device, d)
            _rows("q_out", q_out, self.device, d)
            _need(q.dtype == k.dtype and q.shape == q_out.shape and q.shape[0] == k.shape[0],
                  "q must have the rows and type of k, and q_out the shape of q")
            _written("q_out", q_out)
            _need(q_out.data_ptr() != q.data_ptr() or (q_out.dtype == q.dtype and _strides(q_out) == _strides(q)),
                  "q_out may be q only with its dtype and strides")
            heads, out_dtype = q.shape[1], q_out.dtype
        length = 0
        if cos is not None:
            _need(cos.dim() == 2, "cos and sin must be [positions, head dim / 2]")
            length = cos.shape[0]
        args = _core.KV8AppendArgs(
            ctypes.sizeof(_core.KV8AppendArgs), _TYPES[k.dtype], _TYPES[out_dtype], heads, length, 0,
            q.data_ptr() if heads else None, k.data_ptr(), v.data_ptr(), q_out.data_ptr() if heads else None,
            *(_strides(q) if heads else (0, 0)), *_strides(k), *_strides(v),
            *(_strides(q_out) if heads else (0, 0)),
            _vector("q_norm", q_norm, self.device, (d,)), _vector("k_norm", k_norm, self.device, (d,)),
            _vector("cos", cos, self.device, (length, d // 2)), _vector("sin", sin, self.device, (length, d // 2)))
        return KV8Call(_core.lib().mg_kv8_append, batch, (self._c, self._batch(batch, k.shape[0]), args),
                       (self, q, k, v, q_out, q_norm, k_norm, cos, sin))

    def append(self, batch: KV8Batch, k: torch.Tensor, v: torch.Tensor, **more: Any) -> None:
        """``append_call`` with the same arguments, launched once."""
        self.append_call(batch, k, v, **more)()

    # --------------------------------------------------------------- attention
    def workspace_bytes(self, batch: KV8Batch, heads: int) -> int:
        """Bytes of workspace that an attention call with these bounds needs."""
        n = ctypes.c_int64()
        with torch.cuda.device(self.device):
            _core._check(_core.lib().mg_kv8_attention_workspace(  # noqa: SLF001
                ctypes.byref(self._c), ctypes.byref(self._batch(batch, 1)), heads, ctypes.byref(n)))
        return n.value

    def attention_call(self, batch: KV8Batch, q: torch.Tensor, out: torch.Tensor, *, scale: float | None = None,
                       window: int = 0, workspace: torch.Tensor | None = None) -> KV8Call:
        """Binds ``mg_kv8_attention``: q and out [rows, heads, head dim], bfloat16 or float16 (which an append of float32
        rows may write as its q_out); scale defaults to head_dim ** -0.5; window 0:
        every earlier position.  workspace: a uint8 tensor of at least ``workspace_bytes``."""
        d = self.head_dim
        _rows("q", q, self.device, d)
        _rows("out", out, self.device, d)
        _need(q.shape == out.shape and q.dtype == out.dtype, "out must have the shape and type of q")
        _written("out", out)
        _need(q.data_ptr() != out.data_ptr(), "out must not be q")
        size = self.workspace_bytes(batch, q.shape[1])
        own: tuple[torch.Tensor, ...] = ()
        if workspace is None:
            workspace = torch.empty(size, dtype=torch.uint8, device=self.device)
            own = (workspace,)
        _need(workspace.dtype == torch.uint8 and workspace.device == self.device and workspace.is_contiguous(),
              f"workspace must be a contiguous uint8 tensor on {self.device}")
        args = _core.KV8AttentionArgs(
            ctypes.sizeof(_core.KV8AttentionArgs), _TYPES[q.dtype], q.shape[1], _i32(window),
            d ** -0.5 if scale is None else float(scale), 0, q.data_ptr(), out.data_ptr(), *_strides(q),
            *_strides(out), workspace.data_ptr(), workspace.numel())
        return KV8Call(_core.lib().mg_kv8_attention, batch, (self._c, self._batch(batch, q.shape[0]), args),
                       (self, q, out, workspace), own)

    def attention(self, batch: KV8Batch, q: torch.Tensor, out: torch.Tensor | None = None, **more: Any) -> torch.Tensor:
        """``attention_call`` with the same arguments, launched once; returns out (a new tensor if none is given)."""
        if out is None:
            out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        self.attention_call(batch, q, out, **more)()
        return out
