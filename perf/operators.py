"""Measured cases of the 8-bit paged cache: appending keys and values, and the attention that reads them.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits, 64 where a value may lie next to a rounding border), or, with
``own`` set, through the package's own calls.  ``exact`` restates the same
definitions sequence by sequence in 64 bits.

The cache holds e4m3 codes in pages ``[pages, kv heads, page size, head dim]``
with one fp32 scale per 16 tokens and kv head; a sequence's page list is its
row of the page table.  The new tokens of all sequences are packed by rows,
``q_start[b] .. q_start[b + 1]``; ``ctx_len[b]`` counts sequence b's positions
with them.
"""

import math
import random

import torch

own = False

BLOCK = 16  # tokens per scale
E4M3_MAX = 448.0
EPS = 1e-6
THETA = 1e6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    one_b = {"heads": 4, "kv_heads": 1, "dim": 256}    # Gemma3-1B
    four_b = {"heads": 8, "kv_heads": 4, "dim": 256}   # Gemma3-4B
    big = {"heads": 32, "kv_heads": 16, "dim": 128}    # Gemma3-27B
    return [
        # one stream of the 1B model stores its next token: latency
        _case("append-1b-one-token", "append", one_b, type="bf16", page=16, batch=1, q=1, ctx=640, norm=True),
        # a full serving batch of the 27B model, one token each, into partly filled blocks
        _case("append-27b-128-rows", "append", big, type="f16", page=64, batch=128, q=1, ctx=4096, norm=True),
        # prompts of the 4B model straight from the fp32 products of the batched prefill, two of them continuing
        _case("append-4b-prompts", "append", four_b, type="f32", page=32, batch=5, q=1500, ctx=2048, norm=True),
        # one long prompt of the 27B model, no norm weights
        _case("append-27b-long", "append", big, type="bf16", page=64, batch=1, q=16384, ctx=16384, norm=False),
        # one stream of the 1B model in the middle of the benchmark's positions: latency
        _case("attention-1b-one-stream", "attention", one_b, type="bf16", page=16, batch=1, q=1, ctx=640),
        # one stream at the end of a long context: a single sequence and kv head for the whole GPU
        _case("attention-1b-long", "attention", one_b, type="bf16", page=64, batch=1, q=1, ctx=131072),
        # a serving batch of the 4B model on a local layer: 1024 positions each, out of long contexts
        _case("attention-4b-window", "attention", four_b, type="bf16", page=32, batch=96, q=1, ctx=8192, window=1024),
        # a serving batch of the 27B model on a global layer, contexts of many lengths
        _case("attention-27b-batch", "attention", big, type="f16", page=64, batch=32, q=1, ctx=16384),
        # four drafted tokens per stream, checked in one pass
        _case("attention-1b-drafts", "attention", one_b, type="bf16", page=16, batch=24, q=4, ctx=6001),
        # a chunk of a prompt behind a cached prefix (4B)
        _case("attention-4b-chunk", "attention", four_b, type="bf16", page=32, batch=2, q=512, ctx=8192),
        # prompts of the encoder's head size with small heads, ragged
        _case("attention-64-prompts", "attention", {"heads": 12, "kv_heads": 4, "dim": 64}, type="f16", page=16,
              batch=7, q=777, ctx=777),
        # a whole prompt of the 27B model
        _case("attention-27b-prompt", "attention", big, type="bf16", page=64, batch=1, q=4096, ctx=4096),
    ]


def _case(name, op, heads, **more):
    return {"name": name, "op": op, **heads, "window": 0, "norm": False, **more}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        kv = rng.choice([1, 2, 3, 4, 8, 16])
        case = {"op": rng.choice(["append", "attention", "attention"]), "kv_heads": kv,
                "heads": kv * rng.choice([1, 2, 3, 4, 6, 8]), "dim": rng.choice([64, 128, 256]),
                "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "f16"]), "window": 0,
                "norm": False}
        kind = rng.choice(["token", "token", "drafts", "prompt"])
        if kind == "prompt":
            case["batch"] = log(1, 16)
            case["q"] = log(17, 8192)
            case["ctx"] = case["q"] + (log(1, 8192) if rng.random() < 0.5 else 0)
        else:
            case["q"] = 1 if kind == "token" else rng.randint(2, 8)
            case["batch"] = log(1, 256)
            case["ctx"] = log(8, 65536)
        if case["op"] == "append":
            case["type"] = rng.choice(["bf16", "f16", "f32"])
            case["norm"] = rng.random() < 0.5
        elif rng.random() < 0.3:
            case["window"] = log(1, case["ctx"])
        cells = case["batch"] * case["ctx"] * kv * case["dim"]
        scores = case["batch"] * case["heads"] * case["q"] * case["ctx"]
        new = case["batch"] * case["q"] * (case["heads"] + 2 * kv) * case["dim"]
        flops = 4 * scores * case["dim"]
        if case["op"] == "append" and new <= 1.2e8 and cells <= 5e8:
            return case
        if case["op"] == "attention" and cells <= 6e8 and scores <= 5e8 and flops <= 1.3e11:
            return case


def _lens(case):
    """(new tokens, positions with them) of each sequence; the first has the case's own."""
    q, ctx = [], []
    for b in range(case["batch"]):
        f = 1.0 if b == 0 else (b * 0.6180339887498949) % 1.0
        nq = case["q"] if case["q"] <= 8 else max(1, int(case["q"] * (0.25 + 0.75 * f)))
        more = case["ctx"] - case["q"]
        q.append(nq)
        ctx.append(nq + int(more * (0.25 + 0.75 * f)) if more > 0 else nq)
    return q, ctx


def _seen(case):
    """(visible positions that some query of a sequence reads, visible (query, position) pairs), summed over sequences."""
    rows = pairs = 0
    for q, ctx in zip(*_lens(case)):
        w = case["window"] or ctx
        first = max(0, ctx - q + 1 - w)
        rows += ctx - first
        lo, hi = ctx - q + 1, ctx  # positions that a query sees without the window: lo .. hi
        full = max(0, hi - max(lo, w) + 1)
        pairs += w * full + sum(range(lo, min(hi, w - 1) + 1)) if w >= lo else w * q
    return rows, pairs


def work(case):
    hq, hkv, hd = case["heads"], case["kv_heads"], case["dim"]
    q, _ = _lens(case)
    n, size = sum(q), torch.empty(0, dtype=_TYPES[case["type"]]).element_size()
    if case["op"] == "append":
        out = 2 if case["type"] == "f32" else size
        scales = 2 * 4 * hkv * (n / BLOCK + case["batch"])
        return {"bytes": n * hd * (hq * (size + out) + 2 * hkv * (size + 1) + 4) + scales,
                "flops": n * hd * (3 * hq + 5 * hkv)}
    rows, pairs = _seen(case)
    return {"bytes": rows * hkv * (2 * hd + 2 * 4 / BLOCK) + 2 * n * hq * hd * size, "flops": 4 * pairs * hq * hd}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    r = random.Random(seed)
    q, ctx = _lens(case)
    hq, hkv, hd, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    kind, n = _TYPES[case["type"]], sum(q)
    need = [-(-c // page) for c in ctx]
    pages = sum(need) + 3
    order = list(range(pages))
    r.shuffle(order)
    width = max(need) + 1
    table, at = [], 0
    for m in need:
        table.append(order[at:at + m] + [-1] * (width - m))
        at += m

    def cached():
        """Codes of normal values, each block with a scale of its own that fits a value spread of about one."""
        codes = torch.empty(pages, hkv, page, hd, dtype=torch.float8_e4m3fn, device=dev)
        step = max(1, (1 << 27) // (hkv * page * hd))
        for i in range(0, pages, step):
            part = codes[i:i + step]
            part.copy_((torch.randn(part.shape, device=dev, generator=g) * 90.0).clamp_(-E4M3_MAX, E4M3_MAX))
        power = torch.randint(-8, -4, (pages, hkv, page // BLOCK), device=dev, generator=g)
        return codes, torch.exp2(power.float())

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    start = [0]
    for m in q:
        start.append(start[-1] + m)
    s = {"case": case, "q_start": ints(start), "ctx_len": ints(ctx), "table": ints(table), "max_q": max(q),
         "max_ctx": max(ctx)}
    s["k"], s["k_scale"] = cached()
    s["v"], s["v_scale"] = cached()
    if case["op"] == "append":
        # rows as a fused projection leaves them: the q heads, the k heads, the v heads
        qkv = torch.randn(n, hq + 2 * hkv, hd, device=dev, generator=g).to(kind)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_out"] = torch.empty(n, hq, hd, dtype=torch.bfloat16 if kind == torch.float32 else kind, device=dev)
        angle = torch.arange(max(ctx), device=dev, dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = torch.randn(hd, device=dev, generator=g) * 0.2 if case["norm"] else None
        s["k_norm"] = torch.randn(hd, device=dev, generator=g) * 0.2 if case["norm"] else None
    else:
        s["q"] = torch.randn(n, hq, hd, device=dev, generator=g).to(kind)
        s["out"] = torch.empty_like(s["q"])
    if own:  # the program's handle on the cache and its batch, and the call it repeats every step
        from mogemma_b200.kv8 import KV8Batch, KV8Cache

        cache = KV8Cache.wrap(s["k"], s["v"], s["k_scale"], s["v_scale"])
        batch = KV8Batch(s["q_start"], s["ctx_len"], s["table"], max_q=s["max_q"], max_ctx=s["max_ctx"])
        if case["op"] == "append":
            s["call"] = cache.append_call(batch, s["new_k"], s["new_v"], q=s["q"], q_out=s["q_out"],
                                          q_norm=s["q_norm"], k_norm=s["k_norm"], cos=s["cos"], sin=s["sin"])
        else:
            s["call"] = cache.attention_call(batch, s["q"], s["out"], scale=hd ** -0.5, window=case["window"])
    return s


def run(state):
    append = state["case"]["op"] == "append"
    if own:
        state["call"]()
    elif append:
        _append(state)
    else:
        state["out"] = _attention(state)
    if append:
        return {"q": state["q_out"], "k": state["k"], "v": state["v"], "k_scale": state["k_scale"],
                "v_scale": state["v_scale"]}
    return state["out"]


# ---------------------------------------------------------------- plain forms
def _padded(state, x):
    """Packed rows as [sequence, new token, ...], and which of them are real."""
    start = state["q_start"].long()
    i = torch.arange(state["max_q"], device=x.device)
    row = start[:-1, None] + i
    real = row < start[1:, None]
    return x[torch.where(real, row, 0)], real


def _positions(state):
    """Position of every packed row."""
    start, ctx = state["q_start"].long(), state["ctx_len"].long()
    row = torch.arange(state["q"].shape[0], device=start.device)
    b = torch.searchsorted(start, row, right=True) - 1
    return ctx[b] - (start[b + 1] - row)


def _turned(x, norm, cos, sin):
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + norm.to(x.dtype))
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos.to(x.dtype)[:, None], sin.to(x.dtype)[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _append(state):
    pos = _positions(state)
    cos, sin = state["cos"][pos], state["sin"][pos]
    state["q_out"].copy_(_turned(state["q"].float(), state["q_norm"], cos, sin))
    _store(state, _turned(state["new_k"].double(), state["k_norm"], cos, sin), state["k"], state["k_scale"])
    _store(state, state["new_v"].double(), state["v"], state["v_scale"])


def _store(state, x, codes, scales):
    """Quantises packed rows x [n, heads, dim] into their blocks; earlier tokens of a block follow a larger scale."""
    dev, page = x.device, state["case"]["page"]
    start, ctx = state["q_start"].long(), state["ctx_len"].long()
    first = ctx - (start[1:] - start[:-1])  # position of each sequence's first new token
    block = first[:, None] // BLOCK + torch.arange((state["max_q"] + BLOCK - 2) // BLOCK + 1, device=dev)
    pos = block[..., None] * BLOCK + torch.arange(BLOCK, device=dev)  # [sequence, block, slot]
    new = (pos >= first[:, None, None]) & (pos < ctx[:, None, None])
    old = pos < first[:, None, None]
    touched = new.any(-1)
    value = x[torch.where(new, start[:-1, None, None] + pos - first[:, None, None], 0)]  # [.., slot, head, dim]
    value = torch.where(new[..., None, None], value, 0.0)
    frac, power = torch.frexp(value.abs().amax((2, 4)))  # [sequence, block, head]
    scale = torch.exp2((power - 9 + (frac > 0.875)).clamp(min=-100).double())
    at = torch.where(touched, block * BLOCK // page, 0)
    pid = torch.where(touched, state["table"].long().gather(1, at), 0)
    sub = block * BLOCK % page // BLOCK
    before = scales[pid, :, sub].double()
    scale = torch.where(old.any(-1, keepdim=True), torch.maximum(scale, before), scale)
    slot = pos % page
    held = codes[pid[..., None], :, slot].double() * (before / scale)[:, :, None, :, None]
    value = torch.where(old[..., None, None], held, value / scale[:, :, None, :, None])
    keep = touched[..., None] & (old | new)
    codes[pid[..., None].expand_as(slot)[keep], :, slot[keep]] = value.float()[keep].to(codes.dtype)
    scales[pid[touched], :, sub[touched]] = scale[touched].float()


def _values(state, codes, scales):
    """The cached values as [sequence, kv head, position, dim] in 32 bits."""
    table = state["table"].long()[:, :-1].clamp(min=0)
    x = codes[table].float() * scales[table].repeat_interleave(BLOCK, 3)[..., None]
    b, p, h, t, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * t, d)


def _attention(state):
    case = state["case"]
    hq, hkv, hd = case["heads"], case["kv_heads"], case["dim"]
    x, real = _padded(state, state["q"])  # [sequence, new token, head, dim]
    b, m = x.shape[:2]
    x = x.float().reshape(b, m, hkv, hq // hkv, hd).transpose(1, 2).reshape(b, hkv, -1, hd)
    score = x @ _values(state, state["k"], state["k_scale"]).transpose(-1, -2) * hd ** -0.5
    start, ctx = state["q_start"].long(), state["ctx_len"].long()
    at = (ctx - (start[1:] - start[:-1]))[:, None] + torch.arange(m, device=ctx.device)
    t = torch.arange(score.shape[-1], device=ctx.device)
    see = t <= at[..., None]
    if case["window"]:
        see &= t > at[..., None] - case["window"]
    see = see.repeat_interleave(hq // hkv, 1)[:, None]
    score = score.masked_fill(~see, -math.inf)
    score = (score - score.amax(-1, keepdim=True)).exp()
    out = (score @ _values(state, state["v"], state["v_scale"])) / score.sum(-1, keepdim=True)
    out = out.reshape(b, hkv, m, hq // hkv, hd).transpose(1, 2).reshape(b, m, hq, hd)
    return out[real].to(state["q"].dtype)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    q_start, ctx, table = s["q_start"].tolist(), s["ctx_len"].tolist(), s["table"].tolist()
    return _exact_append(s, q_start, ctx, table) if case["op"] == "append" else _exact_attention(s, q_start, ctx, table)


def _e4m3(x):
    """Round to nearest even among e4m3 values: 4 significant bits, steps of 2^-9 at the least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s, q_start, ctx, table):
    case = s["case"]
    hd, page = case["dim"], case["page"]

    def turn(x, w, at):
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + EPS) * (w.double() + 1)
        z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * torch.complex(
            s["cos"][at].double(), s["sin"][at].double())[:, None]
        return torch.cat([z.real, z.imag], -1)

    out = {"q": torch.empty_like(s["q"], dtype=torch.float64)}
    for name in ("k", "v"):
        out[name], out[name + "_scale"] = s[name].double(), s[name + "_scale"].double()
    for b, c in enumerate(ctx):
        rows = slice(q_start[b], q_start[b + 1])
        p0 = c - (q_start[b + 1] - q_start[b])
        at = torch.arange(p0, c, device=s["q"].device)
        out["q"][rows] = turn(s["q"][rows].double(), s["q_norm"], at)
        for name, x in (("k", turn(s["new_k"][rows].double(), s["k_norm"], at)), ("v", s["new_v"][rows].double())):
            for blk in range(p0 // BLOCK, (c - 1) // BLOCK + 1):
                lo, hi = max(p0, blk * BLOCK), min(c, (blk + 1) * BLOCK)
                part = x[lo - p0:hi - p0]
                most = part.abs().amax((0, 2))
                scale = torch.exp2(torch.ceil(torch.log2((most / E4M3_MAX).clamp(min=2.0 ** -100))))
                pid, slot, j = table[b][blk * BLOCK // page], blk * BLOCK % page, blk * BLOCK % page // BLOCK
                had = lo - blk * BLOCK
                if had:
                    prev = out[name + "_scale"][pid, :, j].clone()
                    scale = torch.maximum(scale, prev)
                    held = out[name][pid, :, slot:slot + had]
                    held.copy_(_e4m3(held * (prev / scale)[:, None, None]))
                codes = _e4m3(part / scale[:, None]).transpose(0, 1)
                out[name][pid, :, slot + had:slot + had + hi - lo] = codes
                out[name + "_scale"][pid, :, j] = scale
    return out


def _exact_attention(s, q_start, ctx, table):
    case = s["case"]
    group, hd, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.empty_like(s["q"], dtype=torch.float64)
    for b, c in enumerate(ctx):
        ids = torch.tensor(table[b][:-(-c // page)], device=out.device)
        n = q_start[b + 1] - q_start[b]
        rows = slice(q_start[b], q_start[b + 1])
        at = torch.arange(c - n, c, device=out.device)[:, None]
        t = torch.arange(c, device=out.device)
        hide = t > at
        if case["window"]:
            hide |= t <= at - case["window"]
        for h in range(case["kv_heads"]):
            k, v = ((s[name][ids, h].double().reshape(-1, BLOCK, hd)
                     * s[name + "_scale"][ids, h].double().reshape(-1, 1, 1)).reshape(-1, hd)[:c] for name in "kv")
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][rows, j].double() @ k.T) / math.sqrt(hd)
                score[hide] = -math.inf
                out[rows, j] = torch.softmax(score, -1) @ v
    return out
