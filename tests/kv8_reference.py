"""The 8-bit paged cache in 64 bits, sequence by sequence: what the kernels are compared with."""

from __future__ import annotations

import math

import torch

BLOCK = 16
E4M3_HALF_STEP = 2.0**-4  # relative; 2^-10 below the normal range


def rope_tables(length: int, dim: int, device, theta: float = 1e4):
    angle = torch.arange(length, dtype=torch.float64)[:, None] * theta ** (
        -torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def turned(x, norm, cos, sin, pos):
    """rope(norm(x)) of rows x [n, heads, dim] at positions pos, in 64 bits."""
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + norm.double())
    if cos is None:
        return x
    h = x.shape[-1] // 2
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def gather(codes, scales, table, n):
    """A sequence's first n cached values [kv heads, n, dim] in 64 bits."""
    page = codes.shape[2]
    ids = torch.as_tensor(table[: -(-n // page)], dtype=torch.long, device=codes.device)
    c = codes.view(torch.float8_e4m3fn)[ids].double()  # [pages, heads, page, dim]
    c = c * scales[ids].double().repeat_interleave(BLOCK, 2)[..., None]
    return c.transpose(0, 1).flatten(1, 2)[:, :n]


def attention(q, k, v, first, scale, window):
    """softmax(scale q k^T) v and the same over |v|, for queries q [n, heads, dim] at positions first, first + 1, ...

    k, v [kv heads, ctx, dim]; positions of k: 0 .. ctx - 1.  Also the largest sum |scale q k| of a pair."""
    n, heads, _ = q.shape
    group = heads // k.shape[0]
    out, size, most = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0.0
    at = torch.arange(first, first + n, device=q.device)[:, None]
    t = torch.arange(k.shape[1], device=q.device)
    see = t <= at
    if window:
        see &= t > at - window
    for h in range(heads):
        kk, vv, qq = k[h // group], v[h // group], q[:, h].double()
        s = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
        p = torch.where(see.any(-1, keepdim=True), torch.softmax(s, -1), 0.0)
        out[:, h], size[:, h] = p @ vv, p @ vv.abs()
        if k.shape[1]:
            most = max(most, float((qq.abs() @ kk.abs().T * abs(scale)).max()))
    return out, size, most


def attention_tolerance(out, size, most, vmax, seen, dim, dtype):
    """Elementwise bound of the kernels' error.

    Products of fp16-exact operands summed in fp32, at most one rounding (2^-23, truncation included) per term:
    a score is off by 2^-23 (dim + 8) sum |scale q k|; with the exponentials (2 ulp) every probability is off by
    twice that plus 2^-21 relative.  P is rounded to fp16: 2^-11 relative, or 2^-25 of the largest where it
    underflows.  The result is rounded once."""
    delta = 2 * 2.0**-23 * (dim + 8) * most + 2.0**-20
    return (torch.finfo(dtype).eps / 2 * out.abs() + size * (2.0**-11 + 2 * delta) + seen * 2.0**-25 * vmax
            + torch.finfo(dtype).tiny)
