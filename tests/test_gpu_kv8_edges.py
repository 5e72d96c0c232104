"""Edges of mg_kv8_append and mg_kv8_attention on the GPU."""

from __future__ import annotations

import time

import pytest

torch = pytest.importorskip("torch")

import kv8_reference as ref  # noqa: E402

from mogemma_b200.kv8 import KV8Batch, KV8Cache, set_debug  # noqa: E402
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


# ---------------------------------------------------------------- weights far below a row's largest
def _one_hot_world(lens, *, dim, page, codes, kv_heads=1, seed=0):
    """Keys whose score is their first code alone: codes [positions] (shared by sequences), the rest 0; scales of 1."""
    w = World(lens, kv_heads=kv_heads, dim=dim, page=page, seed=seed)
    c = w.cache
    c.k_scale.fill_(1.0)
    c.v_scale.fill_(1.0)
    c.k.view(torch.uint8).zero_()
    for b, (_, ctx) in enumerate(lens):
        for p0 in range(0, ctx, page):
            m = min(page, ctx - p0)
            c.k[w.table[b][p0 // page], :, :m, 0] = codes[p0:p0 + m, None].T.to(c.k.dtype).expand(kv_heads, m)
    return w


def _set_values(w, b, at, row):
    """Sequence b's value at position `at` of every head becomes row."""
    w.cache.v[w.table[b][at // w.page], :, at % w.page] = row.to(w.cache.v.dtype)


# P is rounded to fp16 as 2^lift times its ratio to the row's largest so far
@pytest.mark.parametrize(("n", "dim", "group", "lift"), [
    (1, 256, 4, 15), (1, 64, 1, 15), (6, 128, 2, 15), (40, 64, 1, 8), (70, 128, 2, 8), (20, 256, 4, 8)])
@pytest.mark.parametrize("depth", [18.0, 25.2, 30.0])
def test_a_long_tail_of_small_weights_counts(n, dim, group, lift, depth) -> None:
    """One token whose weight is 2^depth of every other's and whose value is 0, before 100000 equal ones; 600 streams over
    the same pages, so that every CTA meets whole contexts (parts of a context have maxima of their own)."""
    ctx, streams = 100_000, 600
    codes = torch.full((ctx,), -8.0, device="cuda")
    codes[3] = 8.0
    w = _one_hot_world([(n, ctx)], dim=dim, page=256, codes=codes)
    g = torch.Generator(device="cuda").manual_seed(1)
    w.cache.v.copy_(torch.randint(64, 448, (w.cache.v.shape[0], 1, 1, dim), device="cuda", generator=g)
                    .expand(w.cache.v.shape))  # all of a sign: the tail does not cancel
    _set_values(w, 0, 3, torch.zeros(dim, device="cuda"))
    batch = KV8Batch(_ints(range(0, streams * n + 1, n)), _ints([ctx] * streams), _ints(w.table * streams), max_q=n,
                     max_ctx=ctx)
    q = torch.zeros(streams * n, group, dim, dtype=BF16, device="cuda")
    q[..., 0] = 1.0
    scale = depth / 16 / 1.4426950408889634
    out = w.cache.attention(batch, q, scale=scale).view(streams, n, group, dim)
    batch.check()
    k, v = (ref.gather(x, s, w.table[0], ctx) for x, s in ((w.cache.k, w.cache.k_scale), (w.cache.v, w.cache.v_scale)))
    o, size, most = ref.attention(q[:n], k, v, ctx - n, scale, 0)
    delta = 2 * 2.0**-23 * (dim + 8) * most + 2.0**-20
    # below fp16's normal range a half step is 2^-25, relative to the 2^lift that the largest P was at its time
    tol = (torch.finfo(BF16).eps / 2 * o.abs() + size * (2.0**-11 + 2 * delta)
           + ctx * 2.0**(-25 - lift) * float(v.abs().max()) + 2.0**-126)
    worst = float(((out.double() - o).abs() / tol).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(("n", "dim", "group"), [
    (1, 64, 2), (4, 128, 3), (2, 256, 8), (50, 64, 2), (50, 128, 1), (20, 256, 3)])
def test_query_elements_far_below_their_rows_largest(n, dim, group, dtype) -> None:
    """The largest elements meet keys of zero, and the scores come from elements 2^-15 to 2^-31 of them."""
    w = World([(n, 300), (n, 65)], kv_heads=2, dim=dim, page=32, seed=dim)
    w.cache.k.view(torch.uint8)[..., ::4] = 0
    q = w.rand(w.rows, 2 * group, dim)
    bf16 = dtype == BF16
    low = torch.full(q.shape, 15, device="cuda")
    if bf16:
        low = torch.randint(24, 31, q.shape, device="cuda", generator=w.g)
    q = (q.clamp(-3.9, 3.9).abs().clamp(min=1.0).copysign(q) * torch.exp2(-low.float()))  # bits down to 2^-38 of 1
    q[..., ::4] = 1.5 if bf16 else 60000.0
    q = q.to(dtype)
    scale = 2.0**25 if bf16 else 2.0**14
    out = w.cache.attention(w.batch, q, scale=scale)
    _check_attention(w, q, out, scale=scale, window=0)


# ---------------------------------------------------------------- bounded waits
@pytest.fixture
def hook():
    yield set_debug
    set_debug()


HANDOFFS = ["items", "items done", "keys", "keys done", "values", "values done", "queries", "scores", "weights",
            "answers", "scales", "halves", "end"]


@pytest.mark.parametrize(("dim", "handoff"), [  # with two row tiles a row is one thread's: no halves
    (dim, h) for dim in (64, 128, 256) for h in HANDOFFS if h != "halves" or dim == 256])
def test_a_wait_that_runs_out_ends_the_call(dim, handoff, hook) -> None:
    """A hand-off of the prompt kernel that never comes: the call ends within its budget and says so, and the next one
    answers as before.  Items of one unit, six or more to a CTA, so that every hand-off is waited for."""
    w = World([(40, 100)] * 450, kv_heads=2, dim=dim, page=32, seed=7)
    q = w.rand(w.rows, 8, dim, dtype=BF16)
    want = w.cache.attention(w.batch, q)
    w.batch.check()
    hook(20_000_000, HANDOFFS.index(handoff))
    t0 = time.perf_counter()
    w.cache.attention(w.batch, q)
    with pytest.raises(RuntimeError, match="wait ran out"):
        w.batch.check()
    assert time.perf_counter() - t0 < 1.0  # the 20 ms budget, not the default's 2 s, ended the waits
    hook()
    assert torch.equal(w.cache.attention(w.batch, q), want)
    w.batch.check()


@pytest.mark.parametrize("dim", [64, 256])
def test_sequences_without_tokens_do_not_hold_up_the_rest(dim, hook) -> None:
    """Two sequences around thousands without tokens, under a bound of many tiles each: going from one to the other
    takes nobody's wait budget."""
    rows = 256 if dim <= 128 else 128
    empty, max_q = 8190, 131_000 * rows // 256
    w = World([(40, 100), *[(0, 0)] * empty, (40, 77)], kv_heads=64, dim=dim, page=16, max_q=max_q)
    q = w.rand(w.rows, 64, dim, dtype=BF16)
    hook(20_000_000)
    out = w.cache.attention(w.batch, q)
    _check_attention(w, q, out, scale=dim**-0.5, window=0)


# ---------------------------------------------------------------- streams
def test_check_sees_calls_on_every_stream() -> None:
    """A call that waits on another stream while check() is made, and one that follows it there at once."""
    w = World([(1, 100), (1, 100)], kv_heads=1, dim=64, page=16, max_ctx=100)
    q = w.rand(w.rows, 2, 64, dtype=F16)
    w.batch.ctx_len[1] = 101
    call = w.cache.attention_call(w.batch, q, torch.zeros_like(q))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            call()
        with pytest.raises(RuntimeError, match="lengths"):
            w.batch.check()
    w.batch.check()


def _load_kernels(w, q) -> None:
    """A kernel's first launch may wait for the device: everything that a test launches has run before."""
    torch.cuda._sleep(1000)
    torch.full((4096,), 255, dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(torch.cuda.Stream()):
        w.cache.attention(KV8Batch(w.batch.q_start, w.batch.ctx_len, w.batch.page_table, max_q=1, max_ctx=16), q)
    torch.cuda.synchronize()


def test_an_error_word_made_on_a_busy_stream() -> None:
    """The batch is made behind work on one stream, and a call on another stream reports before that work is done."""
    w = World([(1, 100), (1, 100)], kv_heads=1, dim=64, page=16, max_ctx=100)
    q = w.rand(w.rows, 2, 64, dtype=F16)
    out, side = torch.zeros_like(q), torch.cuda.Stream()
    _load_kernels(w, q)
    w.batch.ctx_len[1] = 101
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    batch = KV8Batch(w.batch.q_start, w.batch.ctx_len, w.batch.page_table, max_q=1, max_ctx=100)
    call = w.cache.attention_call(batch, q, out)
    with torch.cuda.stream(side):
        call()
    with pytest.raises(RuntimeError, match="lengths"):
        batch.check()


def test_a_workspace_outlives_its_call_on_another_stream() -> None:
    """The call object goes while its launch on another stream still waits: its workspace is not handed out again."""
    w = World([(1, 3000)], kv_heads=2, dim=128, page=16)
    q = w.rand(w.rows, 4, 128, dtype=BF16)
    want, out, side = w.cache.attention(w.batch, q), torch.zeros_like(q), torch.cuda.Stream()
    call = w.cache.attention_call(w.batch, q, out)
    size, places = w.cache.workspace_bytes(w.batch, 4), {call._keep[-1].data_ptr()}
    _load_kernels(w, q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        call()
    del call
    again = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert not places & {x.data_ptr() for x in again}
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_a_call_bound_on_one_stream_and_captured_on_another() -> None:
    w = World([(1, 3000)], kv_heads=2, dim=128, page=16)
    q = w.rand(w.rows, 4, 128, dtype=BF16)
    want, out = w.cache.attention(w.batch, q), torch.zeros_like(q)
    call = w.cache.attention_call(w.batch, q, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call()
    for side in (torch.cuda.current_stream(), torch.cuda.Stream()):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out.zero_()
            graph.replay()
            call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_caches_whose_vectors_share_memory_are_refused() -> None:
    codes = torch.zeros(40_000, dtype=torch.uint8, device="cuda")
    scales = [torch.ones(3, 2, 2, device="cuda") for _ in range(2)]
    shape = (3, 2, 32, 64)
    k, v = (codes[i:].as_strided(shape, (5120, 2560, 80, 1)) for i in (0, 18_448))
    for strides in ((4096, 2048, 64), (4096, 64, 128), (2048, 6144, 64), (5120, 2560, 80)):
        KV8Cache.wrap(*(x.as_strided(shape, (*strides, 1), x.storage_offset()) for x in (k, v)), *scales)
    for strides in ((64, 2048, 64), (4096, 2048, 48), (4096, 64, 64), (4096, 1024, 64), (4096, 0, 64), (0, 2048, 64)):
        with pytest.raises(ValueError, match="must not overlap"):
            KV8Cache.wrap(*(x.as_strided(shape, (*strides, 1), x.storage_offset()) for x in (k, v)), *scales)
    for args in ((k, k, *scales), (k, v, scales[0], scales[0])):
        with pytest.raises(ValueError, match="same memory"):
            KV8Cache.wrap(*args)


# ---------------------------------------------------------------- bad pages and lengths
def _check_rows(w, b, q, out, hidden=()) -> None:
    """Sequence b's answers, query by query, without the positions of the pages in `hidden`."""
    n, ctx = w.lens[b]
    dim = w.cache.head_dim
    table = [w.table[b][0] if i in hidden else p for i, p in enumerate(w.table[b])]
    k, v = (ref.gather(x, s, table, ctx) for x, s in ((w.cache.k, w.cache.k_scale), (w.cache.v, w.cache.v_scale)))
    for i in range(n):
        row, pos = w.start[b] + i, ctx - n + i
        keep = [t for t in range(pos + 1) if t // w.page not in hidden]
        if not keep:
            assert bool((out[row] == 0).all())
            continue
        o, size, most = ref.attention(q[row:row + 1], k[:, keep], v[:, keep], len(keep) - 1, dim**-0.5, 0)
        tol = ref.attention_tolerance(o, size, most, float(v.abs().max()), len(keep), dim, out.dtype)
        assert bool(((out[row:row + 1].double() - o).abs() <= tol).all()), i


@pytest.mark.parametrize(("dim", "page"), [(64, 16), (128, 32), (256, 128)])
@pytest.mark.parametrize("n", [1, 9, 60])
@pytest.mark.parametrize("ids", [(-1, 10**6), (-2**31, 2**31 - 1)])
def test_attention_sees_none_of_a_bad_page(n, dim, page, ids) -> None:
    """One sequence's first and third page are out of range, another's all."""
    w = World([(n, 300), (n, 260), (n, 60), (n, 300)], kv_heads=2, dim=dim, page=page)
    q = w.rand(w.rows, 4, dim, dtype=F16)
    good = w.cache.attention(w.batch, q)
    w.batch.check()
    w.batch.page_table[1, 0], w.batch.page_table[1, 2] = ids
    w.batch.page_table[2] = w.cache.num_pages
    out = w.cache.attention(w.batch, q)
    with pytest.raises(RuntimeError, match="page id"):
        w.batch.check()
    assert torch.equal(out[:n], good[:n]) and torch.equal(out[3 * n:], good[3 * n:])
    _check_rows(w, 1, q, out, hidden=(0, 2))
    assert bool((out[2 * n:3 * n] == 0).all())


def _append_args(w, group, dtype=F32):
    kv, d = w.cache.kv_heads, w.cache.head_dim
    q, k, v = (w.rand(w.rows, h, d, dtype=dtype) for h in (kv * group, kv, kv))
    cos, sin = ref.rope_tables(320, d, "cuda")
    return k, v, {"q": q, "q_out": torch.full_like(q, 7.0), "cos": cos, "sin": sin}


def _restore(w, was) -> None:
    for x, old in zip((w.cache.k, w.cache.v, w.cache.k_scale, w.cache.v_scale), was):
        x.copy_(old)


# max_q chooses the form: a group per token, blocks by sequence, blocks by rows
@pytest.mark.parametrize(("n", "max_q"), [(1, 1), (1, 40), (40, 40), (40, 4000)])
@pytest.mark.parametrize("bad", [-1, -2**31, "num_pages", 2**31 - 1])
def test_append_writes_nothing_for_a_bad_page(n, max_q, bad) -> None:
    w = World([(n, 100), (n, 100), (n, 77)], kv_heads=2, dim=64, page=16, max_q=max_q)
    k, v, more = _append_args(w, 2)
    before = _snapshot(w)
    w.cache.append(w.batch, k, v, **more)
    w.batch.check()
    good, q_out = _snapshot(w), more["q_out"].clone()
    _restore(w, before)
    last = w.table[1][99 // 16]  # the page of the second sequence's last token
    w.batch.page_table[1, 99 // 16] = w.cache.num_pages if bad == "num_pages" else bad
    w.cache.append(w.batch, k, v, **more)
    with pytest.raises(RuntimeError, match="page id"):
        w.batch.check()
    for got, want, old in zip(_snapshot(w), good, before):
        want[last] = old[last]
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(more["q_out"], q_out)  # the queries need no page


@pytest.mark.parametrize(("n", "max_q"), [(1, 1), (1, 40), (40, 40), (40, 4000)])
@pytest.mark.parametrize("ctx", [-5, -2**31, 0, "short", "long", 2**31 - 1])
def test_append_leaves_a_sequence_of_bad_lengths_alone(n, max_q, ctx) -> None:
    w = World([(n, 100), (n, 100), (n, 77)], kv_heads=2, dim=64, page=16, max_q=max_q, max_ctx=100)
    k, v, more = _append_args(w, 2)
    before = _snapshot(w)
    w.cache.append(w.batch, k, v, **more)
    w.batch.check()
    good, q_out = _snapshot(w), more["q_out"].clone()
    _restore(w, before)
    more["q_out"].fill_(7.0)
    w.batch.ctx_len[1] = {"short": n - 1, "long": 101}.get(ctx, ctx)
    w.cache.append(w.batch, k, v, **more)
    with pytest.raises(RuntimeError, match="lengths"):
        w.batch.check()
    mine = w.table[1][:7]
    for got, want, old in zip(_snapshot(w), good, before):
        want[mine] = old[mine]
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    q_out[n:2 * n] = 7.0
    assert torch.equal(more["q_out"], q_out)


@pytest.mark.parametrize("start", [[0, 30, 71, 90], [0, 30, 60, 91], [-1, 30, 60, 90]])
@pytest.mark.parametrize("max_q", [40, 4000])
def test_starts_out_of_bounds_hide_their_own_sequence(start, max_q) -> None:
    """A sequence longer than max_q, one that ends behind the rows, one that starts before them: reported, and the
    sequences before and behind are stored and answered."""
    lens = [(b - a, 100) for a, b in zip(start, start[1:])]
    w = World([(30, 100)] * 3, kv_heads=2, dim=64, page=16, max_q=max_q, max_ctx=100)
    if start[2] == 71:
        w.batch.max_q = 40
    k, v, more = _append_args(w, 2, F16)
    before = _snapshot(w)
    w.batch.q_start.copy_(_ints(start))
    bad = next(i for i, (a, b) in enumerate(zip(start, start[1:])) if a < 0 or b > 90 or b - a > 40)
    w.cache.append(w.batch, k, v, **more)
    with pytest.raises(RuntimeError, match="lengths"):
        w.batch.check()
    out = w.cache.attention(w.batch, more["q_out"])
    with pytest.raises(RuntimeError, match="lengths"):
        w.batch.check()
    for x, old in zip((w.cache.k, w.cache.v, w.cache.k_scale, w.cache.v_scale), before):
        assert torch.equal(x.view(torch.uint8)[w.table[bad][:7]], old.view(torch.uint8)[w.table[bad][:7]])
    w.lens, w.start = lens, start
    for b in range(3):
        if b == bad:
            rows = slice(max(start[b], 0), min(start[b + 1], 90, max(start[b], 0) + w.batch.max_q))
            assert bool((out[rows] == 0).all()) and bool((more["q_out"][rows] == 7.0).all())
        else:
            _check_rows(w, b, more["q_out"], out)
            pos = torch.arange(100 - lens[b][0], 100, device="cuda")
            rows = slice(start[b], start[b + 1])
            got = ref.gather(w.cache.v, w.cache.v_scale, w.table[b], 100)[:, pos].transpose(0, 1)
            near = ref.E4M3_HALF_STEP * v[rows].double().abs() + 2.0**-15  # scales of 2^-5 at most
            assert bool(((got - v[rows].double()).abs() <= near).all()) and bool((more["q_out"][rows] != 7.0).any())


# ---------------------------------------------------------------- far apart
@pytest.mark.parametrize(("n", "dim", "group", "window"), [
    (1, 64, 1, 0), (1, 256, 4, 0), (3, 128, 3, 0), (40, 64, 2, 0), (20, 256, 2, 0),
    (1, 128, 2, 70_001), (33, 128, 1, 70_001)])
def test_attention_over_300000_positions(n, dim, group, window) -> None:
    w = World([(n, 300_001), (n, 131_072)], kv_heads=1, dim=dim, page=128, seed=2)
    q = w.rand(w.rows, group, dim, dtype=BF16)
    out = w.cache.attention(w.batch, q, window=window)
    _check_attention(w, q, out, scale=dim**-0.5, window=window)


@pytest.mark.parametrize("n", [1, 40])
def test_offsets_beyond_32_bits(n) -> None:
    """Pages behind 2^32 bytes of codes, and rows 2^31 elements apart."""
    dim, kv_heads, heads, page, pages = 256, 4, 8, 256, 20_000
    w = World([(n, 700), (n, 900)], kv_heads=kv_heads, dim=dim, page=page)
    far = [torch.empty(pages, kv_heads, page, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
           for _ in range(2)]
    scales = [torch.empty(pages, kv_heads, page // 16, device="cuda") for _ in range(2)]
    move = pages - w.cache.num_pages
    for new, old in zip((*far, *scales), (w.cache.k, w.cache.v, w.cache.k_scale, w.cache.v_scale)):
        new[move:] = old
    w.table = [[p + move if p >= 0 else p for p in t] for t in w.table]
    w.batch.page_table.copy_(_ints(w.table))
    w.cache = KV8Cache.wrap(*far, *scales)
    before = [x[move:].clone() for x in (*far, *scales)]
    # two rows at the ends of a long tensor each, or all of them near its start
    step = 2**31 if w.rows == 2 else 4 * heads * dim
    room = torch.empty(step * (w.rows - 1) + 4 * heads * dim, dtype=BF16, device="cuda")
    at = [room[i * heads * dim:].as_strided((w.rows, h, dim), (step, dim, 1))
          for i, h in enumerate((heads, heads, kv_heads, kv_heads))]
    q, out, k, v = at
    for x in (q, k, v):
        x.copy_(w.rand(*x.shape))
    was = q.clone()
    cos, sin = ref.rope_tables(900, dim, "cuda")
    w.cache.append(w.batch, k, v, q=q, q_out=q, cos=cos, sin=sin)
    near = World(w.lens, kv_heads=kv_heads, dim=dim, page=page)  # the same cache, close at hand
    q2 = was.clone()
    near.cache.append(near.batch, k.contiguous(), v.contiguous(), q=q2, q_out=q2, cos=cos, sin=sin)
    w.batch.check()
    assert torch.equal(q, q2)
    for x, y, old in zip((*far, *scales), (near.cache.k, near.cache.v, near.cache.k_scale, near.cache.v_scale), before):
        assert torch.equal(x[move:].view(torch.uint8), y.view(torch.uint8))
        assert not torch.equal(y.view(torch.uint8), old.view(torch.uint8))
    w.cache.attention(w.batch, q, out)
    _check_attention(w, q, out, scale=dim**-0.5, window=0)


@pytest.mark.parametrize(("n", "dim"), [(1, 64), (1, 256), (8, 128), (40, 64), (40, 256)])
@pytest.mark.parametrize("power", [-120, -100, 100, 118])
def test_value_scales_near_the_ends_of_the_range(n, dim, power) -> None:
    w = World([(n, 300), (n, 65)], kv_heads=2, dim=dim, page=32)
    w.cache.v_scale.fill_(2.0**power)
    q = w.rand(w.rows, 4, dim, dtype=BF16)
    out = w.cache.attention(w.batch, q)
    _check_attention(w, q, out, scale=dim**-0.5, window=0)
    assert bool((out != 0).any())


@pytest.mark.parametrize(("n", "dim"), [(1, 64), (8, 128), (2, 256), (40, 64), (40, 256)])
def test_query_rows_of_subnormals(n, dim) -> None:
    """bf16 rows below 2^-126, brought back by the scale; fp16 rows below 2^-14."""
    w = World([(n, 300), (n, 65)], kv_heads=2, dim=dim, page=32)
    for dtype, power in ((BF16, 129), (F16, 20)):
        q = (w.rand(w.rows, 4, dim) * 2.0**-power).to(dtype)
        scale = 2.0**(power - 3)
        out = w.cache.attention(w.batch, q, scale=scale)
        _check_attention(w, q, out, scale=scale, window=0)


@pytest.mark.parametrize(("n", "dim", "group"), [(600, 64, 1), (600, 128, 2), (300, 256, 2), (1, 128, 4), (5, 256, 2)])
def test_a_non_finite_token_far_behind(n, dim, group) -> None:
    """Where whole units are seen: every query from the token on answers NaN, also long after it, and no other."""
    w = World([(n, 900), (n, 700)], kv_heads=2, dim=dim, page=64)
    q, bad = w.rand(w.rows, 2 * group, dim, dtype=BF16), 450
    good = w.cache.attention(w.batch, q)
    w.cache.k.view(torch.uint8)[w.table[0][bad // 64], 1, bad % 64] = 0x7F  # as the append stores it: K NaN, V 0
    w.cache.v.view(torch.uint8)[w.table[0][bad // 64], 1, bad % 64] = 0
    out = w.cache.attention(w.batch, q)
    windowed = w.cache.attention(w.batch, q, window=100)
    w.batch.check()
    first = max(0, bad - (900 - n))  # the first row that sees it
    assert bool(out[first:n, group:].isnan().all())
    assert torch.equal(out[:first], good[:first]) and torch.equal(out[n:], good[n:])
    assert torch.equal(out[:n, :group], good[:n, :group])
    for i in (first, first + 99, first + 100, n - 1):
        if i < n:
            sees = bad <= 900 - n + i < bad + 100
            assert bool(windowed[i, group:].isnan().all() if sees else windowed[i, group:].isfinite().all())
    assert bool(windowed[n:].isfinite().all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize(("n", "group"), [(1, 33), (1, 128), (3, 100), (7, 128), (1, 17), (2, 13)])
def test_many_heads_to_a_kv_head(dim, n, group) -> None:
    w = World([(n, 500), (n, 31), (n, 129)], kv_heads=1, dim=dim, page=16)
    q = w.rand(w.rows, group, dim, dtype=F16)
    out = w.cache.attention(w.batch, q, window=200)
    _check_attention(w, q, out, scale=dim**-0.5, window=200)


def test_layers_share_one_workspace() -> None:
    """Calls that follow each other, of both kernels and several head dims, over one workspace, eager and in a graph."""
    worlds = [World([(n, 700), (n, 3001)], kv_heads=2, dim=dim, page=32, seed=i)
              for i, (n, dim) in enumerate([(1, 128), (40, 64), (1, 256), (50, 256), (7, 128)])]
    qs = [w.rand(w.rows, 8, w.cache.head_dim, dtype=BF16) for w in worlds]
    want = [w.cache.attention(w.batch, q) for w, q in zip(worlds, qs)]
    size = max(w.cache.workspace_bytes(w.batch, 8) for w in worlds)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    outs = [torch.zeros_like(q) for q in qs]
    calls = [w.cache.attention_call(w.batch, q, o, workspace=ws) for w, q, o in zip(worlds, qs, outs)]
    for call in calls:
        call()
    assert all(torch.equal(o, x) for o, x in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            call()
    for _ in range(5):
        for o in outs:
            o.zero_()
        graph.replay()
        assert all(torch.equal(o, x) for o, x in zip(outs, want))


@pytest.mark.parametrize("max_q", [1, 7, 40, 4000])
def test_a_step_without_tokens_touches_nothing(max_q) -> None:
    """Every sequence idle, though the row tensors have rows (a captured step between two requests)."""
    w = World([(0, 100), (0, 0), (0, 33)], kv_heads=2, dim=64, page=16, extra_rows=5, max_q=max_q)
    k, v, more = _append_args(w, 2, F16)
    before, out = _snapshot(w), w.rand(w.rows, 4, 64, dtype=F16)
    was = out.clone()
    w.cache.append(w.batch, k, v, **more)
    w.cache.attention(w.batch, more["q"], out)
    w.batch.check()
    assert torch.equal(out, was) and bool((more["q_out"] == 7.0).all())
    for x, old in zip(_snapshot(w), before):
        assert torch.equal(x.view(torch.uint8), old.view(torch.uint8))
