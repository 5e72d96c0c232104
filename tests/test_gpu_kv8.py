"""mg_kv8_append and mg_kv8_attention against the 64-bit restatement in kv8_reference.py."""

from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import kv8_reference as ref  # noqa: E402

from mogemma_b200.kv8 import KV8Batch, KV8Cache  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class World:
    """A cache with random contents, sequences with (new tokens, positions), shuffled pages and spare ones."""

    def __init__(self, lens, *, kv_heads, dim, page, seed=0, extra_rows=0, max_q=None, max_ctx=None, layout="heads"):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page = lens, page
        need = [-(-c // page) for _, c in lens]
        pages = sum(need) + 2
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        width = max(1, *need) + 1
        self.table, at = [], 0
        for m in need:
            self.table.append(order[at:at + m] + [-1] * (width - m))
            at += m
        shape = (pages, kv_heads, page, dim) if layout == "heads" else (pages, page, kv_heads, dim)
        codes = [(torch.randn(shape, device="cuda", generator=self.g) * 80).clamp(-448, 448).to(torch.float8_e4m3fn)
                 for _ in range(2)]
        if layout != "heads":
            codes = [c.transpose(1, 2) for c in codes]
        scales = [torch.exp2(torch.randint(-9, -4, (pages, kv_heads, page // 16), device="cuda",
                                           generator=self.g).float()) for _ in range(2)]
        self.cache = KV8Cache.wrap(*codes, *scales)
        self.start = [0]
        for n, _ in lens:
            self.start.append(self.start[-1] + n)
        self.rows = self.start[-1] + extra_rows
        self.batch = KV8Batch(_ints(self.start), _ints([c for _, c in lens]), _ints(self.table),
                              max_q=max_q or max(1, *(n for n, _ in lens)), max_ctx=max_ctx or max(1, *(c for _, c in lens)))

    def rand(self, *shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=self.g) * scale).to(dtype)


def _check_attention(w, q, out, *, scale, window, untouched=None):
    torch.cuda.synchronize()
    c = w.cache
    assert int(w.batch.err.item()) == 0
    for b, (n, ctx) in enumerate(w.lens):
        rows = slice(w.start[b], w.start[b + 1])
        if n == 0:
            continue
        k, v = (ref.gather(x, s, w.table[b], ctx) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
        o, size, most = ref.attention(q[rows], k, v, ctx - n, scale, window)
        vmax = float(v.abs().max()) if ctx else 0.0
        tol = ref.attention_tolerance(o, size, most, vmax, min(ctx, window or ctx), c.head_dim, out.dtype)
        worst = ((out[rows].double() - o).abs() / tol).max()
        assert float(worst) <= 1.0, f"sequence {b} (q {n}, ctx {ctx}): {float(worst):.3g} of the tolerance"
    if untouched is not None:
        assert torch.equal(out[w.start[-1]:], untouched[w.start[-1]:])


# (new tokens, positions) per sequence
ONE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 777)]
MIXED = [(1, 300), (0, 40), (5, 5), (33, 70), (0, 0), (2, 1200), (130, 130)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("dim", "kv_heads", "group", "page"), [
    (64, 2, 1, 16), (64, 1, 8, 128), (128, 3, 2, 32), (128, 2, 9, 64), (256, 1, 4, 16), (256, 2, 3, 256)])
@pytest.mark.parametrize("lens", [ONE, MIXED], ids=["one", "mixed"])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_attention_matches_64_bits(dtype, dim, kv_heads, group, page, lens, window) -> None:
    w = World(lens, kv_heads=kv_heads, dim=dim, page=page, seed=dim + group, extra_rows=3)
    q = w.rand(w.rows, kv_heads * group, dim, dtype=dtype)
    out = w.rand(w.rows, kv_heads * group, dim, dtype=dtype)
    before = out.clone()
    w.cache.attention(w.batch, q, out, window=window)
    _check_attention(w, q, out, scale=dim**-0.5, window=window, untouched=before)


@pytest.mark.parametrize(("dim", "kv_heads", "group", "lens"), [
    (256, 1, 4, [(1, 20011)]), (128, 16, 2, [(1, c) for c in range(900, 3000, 131)]),
    (64, 4, 4, [(3, 5000), (1, 100), (2, 17)]), (256, 2, 2, [(700, 1500)]), (128, 4, 2, [(257, 257), (1, 4096)])])
def test_attention_over_long_contexts(dim, kv_heads, group, lens) -> None:
    w = World(lens, kv_heads=kv_heads, dim=dim, page=64, seed=5)
    q = w.rand(w.rows, kv_heads * group, dim, dtype=BF16)
    out = w.cache.attention(w.batch, q, scale=0.1)
    _check_attention(w, q, out, scale=0.1, window=0)


def test_attention_strides_and_token_major_pages() -> None:
    """Heads between tokens in the pages, q a slice of a fused row, out head major."""
    w = World(MIXED, kv_heads=2, dim=128, page=32, layout="tokens")
    fused = w.rand(w.rows, 10, 128, dtype=F16)
    q = fused[:, 2:8]
    out = torch.zeros(6, w.rows, 128, dtype=F16, device="cuda").transpose(0, 1)
    w.cache.attention(w.batch, q, out, window=90)
    _check_attention(w, q, out, scale=128**-0.5, window=90)


@pytest.mark.parametrize("lens", [[(1, 500), (1, 33)], [(40, 500), (20, 33)]], ids=["token", "chunk"])
def test_attention_scales_far_apart(lens) -> None:
    """Value scales from 2^-40 to 2^40, neighbours 2^30 apart; key scales that make the softmax one-sided."""
    w = World(lens, kv_heads=2, dim=64, page=16)
    c = w.cache
    c.v_scale.copy_(torch.exp2(torch.randint(-4, 5, c.v_scale.shape, device="cuda", generator=w.g).float() * 10))
    c.k_scale.copy_(torch.exp2(torch.randint(-12, 2, c.k_scale.shape, device="cuda", generator=w.g).float()))
    q = w.rand(w.rows, 4, 64, dtype=BF16)
    out = c.attention(w.batch, q, scale=0.02)
    torch.cuda.synchronize()
    for b, (n, ctx) in enumerate(w.lens):
        rows = slice(w.start[b], w.start[b + 1])
        k, v = (ref.gather(x, s, w.table[b], ctx) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
        o, size, most = ref.attention(q[rows], k, v, ctx - n, 0.02, 0)
        # P is held relative to the row's largest probability times scale: compare with that, not with max |V|
        delta = 2 * 2.0**-23 * 72 * most + 2.0**-20
        tol = 2.0**-9 * o.abs() + size * (2.0**-11 + 2 * delta) + ctx * 2.0**-25 * size.amax(-1, keepdim=True) * 448
        assert bool(((out[rows].double() - o).abs() <= tol + 1e-30).all())


@pytest.mark.parametrize("lens", [[(1, 100)], [(50, 100)]], ids=["token", "chunk"])
def test_attention_queries_of_extreme_size(lens) -> None:
    """bf16 rows of 2^100 and 2^-120 (beyond fp16), zero rows, and rows with an infinity or NaN."""
    w = World(lens, kv_heads=1, dim=128, page=16)
    q = w.rand(w.rows, 6, 128, dtype=BF16)
    q[:, 1] = q[:, 1] * 2.0**100
    q[:, 2] = q[:, 2] * 2.0**-120
    q[:, 3] = 0
    q[:, 4, 7] = float("inf")
    q[:, 5, 9] = float("nan")
    out = w.cache.attention(w.batch, q, scale=2.0**-100)
    torch.cuda.synchronize()
    assert bool(out[:, 4:].isnan().all()) and bool(out[:, :4].isfinite().all())
    w2 = out.clone()
    for h in range(4):
        k, v = (ref.gather(x, s, w.table[0], lens[0][1]) for x, s in
                ((w.cache.k, w.cache.k_scale), (w.cache.v, w.cache.v_scale)))
        o, size, most = ref.attention(q[:, h:h + 1], k, v, lens[0][1] - lens[0][0], 2.0**-100, 0)
        tol = ref.attention_tolerance(o, size, most, float(v.abs().max()), lens[0][1], 128, BF16)
        assert bool(((w2[:, h:h + 1].double() - o).abs() <= tol).all()), h


@pytest.mark.parametrize("n", [1, 30])
def test_attention_ignores_what_lies_behind_the_context(n) -> None:
    """Stale NaN codes behind ctx_len, in the same page and block, and pages of -1 behind it."""
    w = World([(n, 45), (n, 64)], kv_heads=2, dim=64, page=64)
    for b, (_, ctx) in enumerate(w.lens):
        p = w.table[b][0]
        for x in (w.cache.k, w.cache.v):
            x.view(torch.uint8)[p, :, ctx:] = 0x7F
    q = w.rand(w.rows, 4, 64, dtype=F16)
    out = w.cache.attention(w.batch, q)
    assert bool(out.isfinite().all())
    _check_attention(w, q, out, scale=0.125, window=0)


@pytest.mark.parametrize("n", [1, 30])
def test_bad_pages_and_lengths_are_reported_and_skipped(n) -> None:
    w = World([(n, 100), (n, 100), (n, 100)], kv_heads=1, dim=64, page=16, max_ctx=100)
    q = w.rand(w.rows, 2, 64, dtype=F16)
    good = w.cache.attention(w.batch, q)
    w.batch.check()
    w.batch.page_table[1, 0] = 10**6
    w.batch.page_table[1, 3] = -7
    out = w.cache.attention(w.batch, q)
    with pytest.raises(RuntimeError, match="page id"):
        w.batch.check()
    assert torch.equal(out[:n], good[:n]) and torch.equal(out[2 * n:], good[2 * n:])
    w.table[1][0] = w.table[1][3] = w.table[1][1]
    k, v = (ref.gather(x, s, w.table[1], 100) for x, s in
            ((w.cache.k, w.cache.k_scale), (w.cache.v, w.cache.v_scale)))
    keep = [t for t in range(100) if t // 16 not in (0, 3)]  # n <= 30: every query sees them all up to its own place
    if n == 1:
        o, size, most = ref.attention(q[n:2 * n], k[:, keep], v[:, keep], len(keep) - 1, 0.125, 0)
        tol = ref.attention_tolerance(o, size, most, float(v.abs().max()), 100, 64, F16)
        assert bool(((out[n:2 * n].double() - o).abs() <= tol).all())
    w.batch.page_table.copy_(_ints(World([(n, 100)] * 3, kv_heads=1, dim=64, page=16).table))
    for bad in ([100, 101, 100], [100, n - 1, 100], [100, -5, 100]):  # beyond max_ctx, shorter than its tokens
        w.batch.ctx_len.copy_(_ints(bad))
        out = w.cache.attention(w.batch, q)
        with pytest.raises(RuntimeError, match="lengths"):
            w.batch.check()
        assert bool((out[n:2 * n] == 0).all())
        assert torch.equal(out[:n], good[:n]) and torch.equal(out[2 * n:], good[2 * n:])


# ---------------------------------------------------------------- append
def _check_append(w, k, v, q, q_out, *, k_norm=None, q_norm=None, cos=None, sin=None, before, before_rows=None):
    """Against the definition: every stored value within half a step of the exact one, the exact scale, earlier
    tokens within half a step of what they were, everything else untouched."""
    torch.cuda.synchronize()
    assert int(w.batch.err.item()) == 0
    c = w.cache
    fp32 = 2.0**-24 * 16  # a norm's sum and scale, a rotation: a few fp32 roundings
    touched = torch.zeros(c.k.shape[:3], dtype=torch.bool, device="cuda")
    scaled = torch.zeros(c.k_scale.shape, dtype=torch.bool, device="cuda")
    for b, (n, ctx) in enumerate(w.lens):
        rows, p0 = slice(w.start[b], w.start[b + 1]), ctx - n
        pos = torch.arange(p0, ctx, device="cuda")
        if q is not None and n:
            want = ref.turned(q[rows], q_norm, cos, sin, pos)
            size = want.abs() + want.abs().roll(c.head_dim // 2, -1)
            tol = torch.finfo(q_out.dtype).eps / 2 * want.abs() + 2 * fp32 * size + torch.finfo(q_out.dtype).tiny
            assert bool(((q_out[rows].double() - want).abs() <= tol).all())
        for x, codes, scales, old_codes, old_scales in (
                (ref.turned(k[rows], k_norm, cos, sin, pos), c.k, c.k_scale, before[0], before[2]),
                (v[rows].double(), c.v, c.v_scale, before[1], before[3])):
            for blk in range(p0 // 16, -(-ctx // 16)) if n else ():
                lo, hi = max(p0, 16 * blk), min(ctx, 16 * blk + 16)
                page, slot = w.table[b][16 * blk // w.page], 16 * blk % w.page
                part = x[lo - p0:hi - p0].transpose(0, 1)
                s = scales[page, :, slot // 16].double()
                need = part.abs().amax((1, 2)) / 448
                want = torch.exp2(torch.ceil(torch.log2(need * (1 - fp32)))).clamp(min=2.0**-100)
                also = torch.exp2(torch.ceil(torch.log2(need * (1 + fp32)))).clamp(min=2.0**-100)
                if lo > 16 * blk:
                    prev = old_scales[page, :, slot // 16].double()
                    want, also = torch.maximum(want, prev), torch.maximum(also, prev)
                    held = old_codes[page, :, slot:slot + lo - 16 * blk].double() * prev[:, None, None]
                    got = codes[page, :, slot:slot + lo - 16 * blk].double() * s[:, None, None]
                    step = torch.maximum(ref.E4M3_HALF_STEP * held.abs(), 2.0**-10 * s[:, None, None])
                    assert bool(((got - held).abs() <= torch.where(s == prev, 0.0, 1.0)[:, None, None] * step).all())
                assert bool(((s == want) | (s == also)).all())
                got = codes[page, :, slot + lo - 16 * blk:slot + hi - 16 * blk].double() * s[:, None, None]
                tol = torch.maximum(ref.E4M3_HALF_STEP * part.abs(), 2.0**-10 * s[:, None, None]) * (1 + 2.0**-16)
                tol = tol + 2 * fp32 * (part.abs() + part.abs().roll(c.head_dim // 2, -1))
                assert bool(((got - part).abs() <= tol).all())
                touched[page, :, slot:slot + hi - 16 * blk] = True
                scaled[page, :, slot // 16] = True
    for new, old in ((c.k, before[0]), (c.v, before[1])):
        assert torch.equal(new.view(torch.uint8)[~touched], old.view(torch.uint8)[~touched])
    for new, old in ((c.k_scale, before[2]), (c.v_scale, before[3])):
        assert torch.equal(new[~scaled], old[~scaled])


def _snapshot(w):
    return [x.clone() for x in (w.cache.k, w.cache.v, w.cache.k_scale, w.cache.v_scale)]


APPEND = [(1, 1), (1, 16), (1, 17), (0, 9), (5, 20), (16, 16), (17, 40), (40, 100), (1, 300), (0, 0), (33, 33)]


@pytest.mark.parametrize(("dtype", "out_dtype"), [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize(("dim", "kv_heads", "group", "page"), [(64, 3, 2, 16), (128, 2, 5, 64), (256, 1, 4, 128)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_matches_64_bits(dtype, out_dtype, dim, kv_heads, group, page, norm) -> None:
    w = World(APPEND, kv_heads=kv_heads, dim=dim, page=page, seed=dim, extra_rows=2)
    qkv = w.rand(w.rows, (group + 2) * kv_heads, dim, dtype=dtype, scale=3.0)
    q, k, v = qkv[:, :group * kv_heads], qkv[:, group * kv_heads:-kv_heads], qkv[:, -kv_heads:]
    q_out = w.rand(w.rows, group * kv_heads, dim, dtype=out_dtype)
    tail = q_out[w.start[-1]:].clone()
    cos, sin = ref.rope_tables(300, dim, "cuda")
    norms = {"q_norm": w.rand(dim, scale=0.3), "k_norm": w.rand(dim, scale=0.3)} if norm else {}
    before = _snapshot(w)
    w.cache.append(w.batch, k, v, q=q, q_out=q_out, cos=cos, sin=sin, **norms)
    _check_append(w, k, v, q, q_out, cos=cos, sin=sin, before=before, **norms)
    assert torch.equal(q_out[w.start[-1]:], tail)


def test_append_in_place_without_rotation_and_token_major_pages() -> None:
    w = World(APPEND, kv_heads=2, dim=128, page=32, layout="tokens", max_q=4000, max_ctx=320)  # blocks found by rows
    q, k, v = (w.rand(w.rows, h, 128, dtype=BF16) for h in (4, 2, 2))
    was, before, wq = q.clone(), _snapshot(w), w.rand(128)
    w.cache.append(w.batch, k, v, q=q, q_out=q, q_norm=wq)
    _check_append(w, k, v, was, q, q_norm=wq, before=before)


def test_append_of_keys_and_values_alone() -> None:
    w = World([(1000, 1203)], kv_heads=4, dim=64, page=16)
    k, v = (w.rand(w.rows, 4, 64, dtype=F32, scale=10.0) for _ in range(2))
    before = _snapshot(w)
    w.cache.append(w.batch, k, v)
    _check_append(w, k, v, None, None, before=before)


def test_append_token_by_token_grows_the_scale() -> None:
    """16 tokens, each twice the size of the last: every append requantises; powers of two lose nothing above
    the subnormal range, and what the block holds stays within its scale's smallest half step."""
    dim, kv_heads = 64, 2
    k, v = (torch.randn(20, kv_heads, dim, device="cuda") for _ in range(2))
    k, v = (x * torch.exp2(torch.arange(20.0, device="cuda"))[:, None, None] for x in (k, v))
    cache = KV8Cache(2, 16, kv_heads, dim)
    for t in range(20):
        batch = KV8Batch(_ints([0, 1]), _ints([t + 1]), _ints([[1, 0]]), max_q=1, max_ctx=32)
        cache.append(batch, k[t:t + 1], v[t:t + 1])
        batch.check()
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        got = ref.gather(codes, scales, [1, 0], 20).transpose(0, 1)
        s = torch.stack([scales[1, :, 0]] * 16 + [scales[0, :, 0]] * 4).double()[..., None]
        # each of up to 15 roundings is exact, or in the subnormal range of the scale of that time: half steps of
        # 2^-10 s, 2^-10 s / 2, ...: together below 2^-9 s
        assert bool(((got - x.double()).abs() <= ref.E4M3_HALF_STEP * x.double().abs() + 2.0**-9 * s).all())


def test_append_of_zeros_and_extremes() -> None:
    w = World([(16, 16), (16, 16), (16, 16)], kv_heads=1, dim=64, page=16)
    k, v = torch.zeros(48, 1, 64, device="cuda"), torch.zeros(48, 1, 64, device="cuda")
    k[16:32], v[16:32] = 1e-35, 3e38
    k[32:, 0, 0], v[32:, 0, 1] = 448.0, 448.00003
    w.cache.append(w.batch, k, v)
    w.batch.check()
    ks, vs = ([float(s[w.table[b][0], 0, 0]) for b in range(3)] for s in (w.cache.k_scale, w.cache.v_scale))
    assert ks == [2.0**-100, 2.0**-100, 1.0] and vs == [2.0**-100, 2.0**120, 2.0]
    v1 = ref.gather(w.cache.v, w.cache.v_scale, w.table[1], 16)
    assert bool(((v1 - 3e38).abs() <= 3e38 * 2.0**-4).all())


def test_a_non_finite_token_poisons_only_those_who_see_it() -> None:
    w = World([(40, 40)], kv_heads=2, dim=64, page=16)
    k, v = (w.rand(40, 2, 64, dtype=F32) for _ in range(2))
    clean_k, clean_v = k.clone(), v.clone()
    k[20, 0, 3], v[25, 1, 5] = float("inf"), float("nan")
    q = w.rand(40, 4, 64, dtype=F16)
    w.cache.append(w.batch, clean_k, clean_v)
    good = w.cache.attention(w.batch, q)
    w.cache.append(w.batch, k, v)
    out = w.cache.attention(w.batch, q)
    windowed = w.cache.attention(w.batch, q, window=4)
    w.batch.check()
    for h, t in ((0, 20), (1, 20), (2, 25), (3, 25)):
        assert bool(out[t:, h].isnan().all()) and bool(out[:t, h].isfinite().all())
        assert bool(windowed[t:t + 4, h].isnan().all())
        assert bool(windowed[:t, h].isfinite().all()) and bool(windowed[t + 4:, h].isfinite().all())
    assert torch.equal(out[:16], good[:16])  # the blocks before theirs are the same


# ---------------------------------------------------------------- together
def test_prompt_then_tokens_as_a_server_runs_them() -> None:
    """Prompts in chunks, then tokens through bound calls captured in a graph, against exact attention over what
    the cache holds, and against attention over the unrounded keys and values."""
    dim, kv_heads, group, page = 128, 2, 2, 16
    heads, total = kv_heads * group, 96
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [60, 33]
    q, k, v = (torch.randn(2, total, h, dim, device="cuda", generator=g).to(BF16) for h in (heads, kv_heads, kv_heads))
    cos, sin = ref.rope_tables(total, dim, "cuda")
    cache = KV8Cache(16, page, kv_heads, dim)
    table = _ints([[3, 1, 5, 7, 9, 11], [0, 2, 4, 6, 8, 10]])

    def answer(b, i0, i1):
        pos = torch.arange(total, device="cuda")
        kk = ref.turned(k[b], None, cos, sin, pos)[:i1].transpose(0, 1)
        qq = ref.turned(q[b], None, cos, sin, pos)[i0:i1]
        return ref.attention(qq, kk, v[b, :i1].double().transpose(0, 1), i0, dim**-0.5, 0)[0]

    done = [0, 0]
    for chunk in (25, 35):  # the second sequence's last chunk is shorter
        n = [min(chunk, m - d) for m, d in zip(lens, done)]
        rows = [torch.cat([x[b, done[b]:done[b] + n[b]] for b in range(2)]) for x in (q, k, v)]
        batch = KV8Batch(_ints([0, n[0], n[0] + n[1]]), _ints([d + m for d, m in zip(done, n)]), table, max_q=40,
                         max_ctx=total)
        cache.append(batch, rows[1], rows[2], q=rows[0], q_out=rows[0], cos=cos, sin=sin)
        out = cache.attention(batch, rows[0])
        batch.check()
        for b, at in ((0, 0), (1, n[0])):
            want = answer(b, done[b], done[b] + n[b])
            err = (out[at:at + n[b]].double() - want).norm() / want.norm()
            assert float(err) < 0.06  # e4m3 keys and values: half steps of 2^-4, averaged
            done[b] += n[b]
    step_q, step_k, step_v = (torch.empty(2, h, dim, dtype=BF16, device="cuda") for h in (heads, kv_heads, kv_heads))
    out = torch.empty_like(step_q)
    ctx = _ints(done)
    batch = KV8Batch(_ints([0, 1, 2]), ctx, table, max_q=1, max_ctx=total)
    append = cache.append_call(batch, step_k, step_v, q=step_q, q_out=step_q, cos=cos, sin=sin)
    attend = cache.attention_call(batch, step_q, out)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.add_(1)
        append()
        attend()
    for _ in range(30):
        for x, step in ((q, step_q), (k, step_k), (v, step_v)):
            step.copy_(torch.stack([x[b, done[b]] for b in range(2)]))
        graph.replay()
        done = [d + 1 for d in done]
        for b in range(2):
            want = answer(b, done[b] - 1, done[b])
            assert float((out[b:b + 1].double() - want).norm() / want.norm()) < 0.09
            kk, vv = (ref.gather(x, s, table[b].tolist(), done[b]) for x, s in
                      ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            o, size, most = ref.attention(step_q[b:b + 1], kk, vv, done[b] - 1, dim**-0.5, 0)
            tol = ref.attention_tolerance(o, size, most, float(vv.abs().max()), done[b], dim, BF16)
            assert bool(((out[b:b + 1].double() - o).abs() <= tol).all())
    batch.check()


def test_the_same_call_gives_the_same_bits() -> None:
    w = World([(1, 5000), (1, 700), (64, 900)], kv_heads=2, dim=128, page=32)
    q = w.rand(w.rows, 8, 128, dtype=BF16)
    first = w.cache.attention(w.batch, q)
    for _ in range(3):
        assert torch.equal(w.cache.attention(w.batch, q), first)


def test_two_streams_with_workspaces_of_their_own() -> None:
    worlds = [World([(1, 3001), (1, 900)], kv_heads=1, dim=256, page=16, seed=s) for s in (1, 2)]
    qs = [w.rand(w.rows, 4, 256, dtype=BF16) for w in worlds]
    want = [w.cache.attention(w.batch, q) for w, q in zip(worlds, qs)]
    outs = [torch.zeros_like(q) for q in qs]
    calls = [w.cache.attention_call(w.batch, q, o) for w, q, o in zip(worlds, qs, outs)]
    streams = [torch.cuda.Stream() for _ in worlds]
    torch.cuda.synchronize()
    for _ in range(20):
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    for got, o in zip(outs, want):
        assert torch.equal(got, o)


def test_bad_tensors_are_refused() -> None:
    w = World([(2, 30), (1, 16)], kv_heads=2, dim=64, page=16)
    c, b = w.cache, w.batch
    q, k, v = (w.rand(w.rows, h, 64, dtype=BF16) for h in (4, 2, 2))
    cos, sin = ref.rope_tables(30, 64, "cuda")
    for call, text in (
            (lambda: c.append(b, k[:, :1], v), "heads"),
            (lambda: c.append(b, k, v.half()), "type"),
            (lambda: c.append(b, k, v, q=q), "together"),
            (lambda: c.append(b, k, v, q=q[:2], q_out=q[:2]), "rows"),
            (lambda: c.append(b, k, v, cos=cos), "cos and sin"),
            (lambda: c.append(b, k, v, cos=cos[:29], sin=sin[:29]), "rope_len"),
            (lambda: c.append(b, k, v, k_norm=torch.ones(32, device="cuda")), "k_norm"),
            (lambda: c.append(b, k.cpu(), v), "on cpu"),
            (lambda: c.append(b, k, v, q=q, q_out=torch.empty(3, 1, 64, dtype=BF16, device="cuda").expand(3, 4, 64)),
             "overlap"),
            (lambda: c.attention(b, q, q.half()), "shape and type"),
            (lambda: c.attention(b, q, q), "must not be q"),
            (lambda: c.attention(b, q.float()), "dtype"),
            (lambda: c.attention(b, q[:, :3]), "multiple"),
            (lambda: c.attention(b, q.transpose(1, 2)), "contiguous"),
            (lambda: c.attention(b, q, workspace=torch.empty(64, dtype=torch.uint8, device="cuda")), "workspace"),
            (lambda: c.attention(b, q, scale=float("nan")), "scale"),
            (lambda: KV8Batch(b.q_start[:2], b.ctx_len, b.page_table, max_q=1, max_ctx=16), "batch . 1"),
            (lambda: KV8Batch(b.q_start.long(), b.ctx_len, b.page_table, max_q=1, max_ctx=16), "int32"),
            (lambda: KV8Cache.wrap(c.k, c.v, c.k_scale[:, :1], c.v_scale), "k_scale"),
            (lambda: KV8Cache.wrap(c.k, c.v[:1], c.k_scale, c.v_scale), "same shape")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            call()
    wide = KV8Batch(b.q_start, b.ctx_len, b.page_table, max_q=2, max_ctx=10**6)
    with pytest.raises(ValueError, match="page table"):
        c.attention(wide, q)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("seed", range(4))
def test_attention_of_items_of_many_sizes(dim, seed) -> None:
    """Sequences whose rows fill one warp, several or all of a row tile, in every order within a CTA's share: what a
    warp skips in one item must not put it out of step in the next."""
    r = random.Random(seed * 3 + dim)
    lens = []
    for _ in range(60):
        n = r.choice([1, 2, 9, 16, 17, 33, 40, 64, 65, 100])
        lens.append((n, n + r.choice([0, 1, 30, 127, 128, 300, 900])))
    w = World(lens, kv_heads=8, dim=dim, page=32, seed=seed)
    q = w.rand(w.rows, 16, dim, dtype=BF16)
    window = r.choice([0, 0, 40, 200])
    out = w.cache.attention(w.batch, q, window=window)
    _check_attention(w, q, out, scale=dim**-0.5, window=window)


@pytest.mark.parametrize("n", [1, 9, 40])
def test_pages_before_the_window_may_be_gone(n) -> None:
    w = World([(n, 700), (n, 333)], kv_heads=2, dim=128, page=16)
    q = w.rand(w.rows, 4, 128, dtype=BF16)
    window = 100
    want = w.cache.attention(w.batch, q, window=window)
    for b, (_, ctx) in enumerate(w.lens):
        w.batch.page_table[b, : (ctx - n + 1 - window) // 16] = -1
    out = w.cache.attention(w.batch, q, window=window)
    w.batch.check()
    assert torch.equal(out, want)


@pytest.mark.parametrize("n", [1, 9, 40])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_negative_and_zero_scales(n, scale) -> None:
    w = World([(n, 200), (n, 77)], kv_heads=2, dim=64, page=32)
    q = w.rand(w.rows, 6, 64, dtype=F16)
    out = w.cache.attention(w.batch, q, scale=scale)
    _check_attention(w, q, out, scale=scale, window=0)


@pytest.mark.parametrize("n", [1, 40])
def test_windows_as_long_as_can_be(n) -> None:
    """A window of 2^31 - 1 is none, also for a sequence whose lengths are refused."""
    w = World([(n, 200), (n, 77)], kv_heads=1, dim=64, page=32)
    q = w.rand(w.rows, 2, 64, dtype=F16)
    want = w.cache.attention(w.batch, q)
    assert torch.equal(w.cache.attention(w.batch, q, window=2**31 - 1), want)
    w.batch.ctx_len[1] = n - 1
    out = w.cache.attention(w.batch, q, window=2**31 - 1)
    with pytest.raises(RuntimeError, match="lengths"):
        w.batch.check()
    assert torch.equal(out[:n], want[:n]) and bool((out[n:] == 0).all())


def test_append_reports_starts_that_fall_back() -> None:
    """The second sequence starts behind its end, in rows that the third one claims; blocks are found by rows."""
    w = World([(60, 60), (50, 50), (60, 60)], kv_heads=1, dim=64, page=64, max_q=1000)
    w.batch.q_start.copy_(_ints([0, 100, 50, 120]))
    k, v = (w.rand(w.rows, 1, 64) for _ in range(2))
    w.cache.append(w.batch, k, v)
    with pytest.raises(RuntimeError, match="lengths"):
        w.batch.check()
