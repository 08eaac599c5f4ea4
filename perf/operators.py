"""The operators of a serving step over a paged KV cache, as a program that serves
several requests at once calls them: the step's plan (block tables, slots and positions
from request lengths), rotary positions with the write into the cache, and attention
of the new tokens over the pages, with or without a sliding window and sinks.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what the program holds, ``run(state)`` is one pass,
``exact(case, seed)`` the outputs from the definition in float64.  With ``own`` false a
pass is elementary torch operations in 32 bits; with ``own`` true it is the calls of
``arcllm_amd``.

Request lengths belong to the case (they are the shape of the work); values, page
orders and free lists come from the seed.  Heads are the 7B shape of the benchmark
(28 query and 4 kv heads of 128) and generic ones.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
RELEASE = -1  # new_lens entry of a finished request: 0xffffffff as int32
NO_SLOT = -1
THETA = 1e6


# ------------------------------------------------------------------- cases
def listed():
    return [
        # every request decodes one token: the plan that precedes each decode step
        dict(name="plan 24 decode", kind="plan", requests=24, chunks=0, chunk=1, ended=2, ctx=3000, page=16, spare=5),
        # a large server's step: most requests decode, some are in their prompt, some have ended
        dict(name="plan 700 mixed", kind="plan", requests=700, chunks=60, chunk=900, ended=25, ctx=9000, page=16,
             spare=100),
        # one decoded token of one request, q|k|v in fp32 as the projection leaves it
        dict(name="rope 1 token", kind="rope", tokens=1, kv_heads=4, hpk=7, dim=128, rot=128, half=0, scaling="plain",
             x="f32", dtype="f16", bias=1, ctx=501, page=16),
        # a ragged step of a long-context configuration: half layout, half of the head, scaled by parts
        dict(name="rope 500 partial scaled", kind="rope", tokens=500, kv_heads=8, hpk=4, dim=128, rot=64, half=1,
             scaling="yarn", x="bf16", dtype="bf16", bias=0, ctx=100000, page=32),
        # a full prompt step
        dict(name="rope 8192 tokens", kind="rope", tokens=8192, kv_heads=4, hpk=7, dim=128, rot=128, half=0,
             scaling="plain", x="f32", dtype="f16", bias=1, ctx=8192, page=16),
        # one request, one token, a short odd context: latency
        dict(name="decode 1 x 501", kind="attn", requests=1, chunks=0, chunk=1, ctx=501, ragged=0, kv_heads=4, hpk=7,
             dim=128, dtype="f16", page=16, window=0, sinks=0),
        # a decode step of many requests with contexts of all lengths
        dict(name="decode 64 x <=8000", kind="attn", requests=64, chunks=0, chunk=1, ctx=8000, ragged=1, kv_heads=4, hpk=7,
             dim=128, dtype="f16", page=16, window=0, sinks=0),
        # two long documents, many shared heads: the context split over the card
        dict(name="decode 2 x 131071", kind="attn", requests=2, chunks=0, chunk=1, ctx=131071, ragged=1, kv_heads=8,
             hpk=8, dim=128, dtype="bf16", page=64, window=0, sinks=0),
        # a mixed step: two requests in their prompt, the others decode
        dict(name="mixed 2 x 512 + 15", kind="attn", requests=17, chunks=2, chunk=512, ctx=5000, ragged=1, kv_heads=8,
             hpk=4, dim=128, dtype="bf16", page=16, window=0, sinks=0),
        # a chunk of a long prompt
        dict(name="chunk 4096 @ 12288", kind="attn", requests=1, chunks=1, chunk=4096, ctx=16384, ragged=0, kv_heads=4,
             hpk=7, dim=128, dtype="f16", page=16, window=0, sinks=0),
        # a windowed layer: decode far behind the window, its first tokens still visible
        dict(name="window decode 48", kind="attn", requests=48, chunks=0, chunk=1, ctx=40000, ragged=1, kv_heads=8, hpk=4,
             dim=128, dtype="bf16", page=32, window=4096, sinks=4),
        # a windowed layer's prompt chunks, heads of 64
        dict(name="window chunks 3 x 2000", kind="attn", requests=3, chunks=3, chunk=2000, ctx=9000, ragged=1, kv_heads=8,
             hpk=8, dim=64, dtype="f16", page=16, window=1024, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "decode", "decode", "chunk", "chunk"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind == "plan":
        B = _log(rng, 1, 1500)
        return dict(kind="plan", requests=B, chunks=rng.randint(0, B // 10 + 1) if B > 1 else 0, chunk=_log(rng, 2, 900),
                    ended=rng.randint(0, B // 8), ctx=_log(rng, 2, 9000), page=page, spare=rng.randint(0, 200))
    heads = dict(kv_heads=rng.choice([1, 2, 3, 4, 5, 8]), hpk=rng.randint(1, 8), dim=rng.choice([64, 128, 128]))
    dtype = rng.choice(["f16", "bf16"])
    if kind == "rope":
        return dict(kind="rope", tokens=_log(rng, 1, 8000), **heads, rot=rng.choice([16, 32, 64, heads["dim"]]),
                    half=rng.randint(0, 1), scaling=rng.choice(["plain", "linear", "yarn", "factors"]),
                    x=rng.choice(["f32", "f32", "f16", "bf16"]), dtype=dtype, bias=rng.randint(0, 1),
                    ctx=_log(rng, 8, 500000), page=page)
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    more = dict(**heads, dtype=dtype, page=page, window=window, sinks=rng.randint(0, 8) if window else 0, ragged=1)
    if kind == "decode":
        B = _log(rng, 1, 96)
        return dict(kind="attn", requests=B, chunks=0, chunk=1, ctx=_log(rng, 1, min(65536, 600000 // B)), **more)
    B, chunk = _log(rng, 1, 12), _log(rng, 2, 1500)
    ctx = chunk + _log(rng, 1, 12000)
    while B > 1 and B * chunk * ctx * heads["kv_heads"] * heads["hpk"] > 1.2e9:
        B -= 1
    return dict(kind="attn", requests=B, chunks=rng.randint(1, B), chunk=chunk, ctx=ctx, **more)


# ------------------------------------------------------------------ lengths
def _lens(c):
    """(positions held before the step, new tokens of the step) of every request."""
    rng = random.Random("%s %s %s %s" % (c.get("requests"), c["ctx"], c.get("chunk"), c.get("chunks")))
    B = c["requests"]
    first = rng.sample(range(B), c["chunks"] + c.get("ended", 0))
    chunks, ended = set(first[: c["chunks"]]), set(first[c["chunks"]:])
    old, new = [], []
    for b in range(B):
        n = 1
        if b in chunks:
            n = c["chunk"] if not c.get("ragged", 1) or c["chunks"] < 3 else rng.randint(max(1, c["chunk"] // 2), c["chunk"])
        most = max(0, c["ctx"] - n)
        held = most if not c.get("ragged", 1) or b == 0 else _log(rng, max(1, most // 40), most) if most else 0
        if c["kind"] == "plan" and b in chunks and rng.random() < 0.6:
            held = 0  # a new request
        old.append(held)
        new.append(RELEASE if b in ended else n)
    return old, new


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------- inputs
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + stream * 7919 + 4242) & 0x7FFFFFFFFFFF)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _layout(g, held, page, free=0):
    """Pages of requests that hold `held` positions, in a random order over the pool:
    (tables [B, longest], free pages, pool size)."""
    need = [_pages(n, page) for n in held]
    total, longest = sum(need), max(1, max(need))
    order = torch.randperm(total + free, generator=g, device=DEV).to(torch.int32)
    need = torch.tensor(need, device=DEV)
    col = torch.arange(longest, device=DEV)[None, :]
    at = (need.cumsum(0) - need)[:, None] + col
    tables = torch.where(col < need[:, None], order[at.clamp(max=max(0, total - 1)).long()], 0).to(torch.int32)
    return tables.contiguous(), order[total:].contiguous(), total + free


def _rot_freqs(c):
    """Angles per position of the rotated pairs (float64, on the CPU), and the factor on
    the rotated values.  linear: positions over 8.  yarn: pairs that turn often within the
    original context keep their angle, slow ones are interpolated by 16, a ramp between.
    factors: an own divisor for each pair."""
    n = c["rot"] // 2
    f = THETA ** (-2.0 * torch.arange(n, dtype=torch.float64) / c["rot"])
    if c["scaling"] == "linear":
        return f / 8.0, 1.0
    if c["scaling"] == "factors":
        return f / _factors(c).double(), 1.0
    if c["scaling"] == "yarn":
        at = lambda turns: c["rot"] * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), c["rot"] - 1)
        ramp = ((torch.arange(n, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / 16.0 * ramp, 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _factors(c):
    return torch.linspace(1.0, 8.0, c["rot"] // 2, dtype=torch.float32)


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    c, g = case, _gen(seed, 0)
    if c["kind"] == "plan":
        e = _prepare_plan(c, g)
    elif c["kind"] == "rope":
        e = _prepare_rope(c, g)
    else:
        e = _prepare_attn(c, g)
    e["c"] = c
    if own:  # the descriptors and workspace that a program of the framework keeps
        e["own"] = _descriptors(e)
    return e


def _prepare_plan(c, g):
    old, new = _lens(c)
    page, B = c["page"], c["requests"]
    taken = sum(_pages(o + n, page) - _pages(o, page) for o, n in zip(old, new) if n != RELEASE)
    tables, free, pool = _layout(g, old, page, taken + c["spare"])
    longest = max(1, max(_pages(o + max(n, 0), page) for o, n in zip(old, new)))
    wide = torch.zeros(B, max(longest, tables.shape[1]), dtype=torch.int32, device=DEV)
    wide[:, : tables.shape[1]] = tables
    stack = torch.zeros(pool, dtype=torch.int32, device=DEV)
    stack[: free.numel()] = free
    tokens = sum(max(n, 0) for n in new)
    rows = tokens + tokens // 16 + 3  # a step's buffers hold some more rows than it uses
    full = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(old=_i32(old), new=_i32(new), tables=wide, stack=stack, count=_i32([free.numel()]), count_out=full(1),
                lens=full(B), starts=full(B + 1), positions=full(rows), slots=full(rows), status=full(4), rows=rows,
                max_new=max(1, max(new)))


def _prepare_rope(c, g):
    N, D, kvh, page = c["tokens"], c["dim"], c["kv_heads"], c["page"]
    heads = kvh * c["hpk"]
    dt, xt = TYPES[c["dtype"]], TYPES[c["x"]]
    cols = (heads + 2 * kvh) * D
    x = (torch.randn(N, cols, generator=g, device=DEV) * 1.5).to(xt)
    # tokens of a few requests at positions all over the context, each in a slot of its own
    pool = _pages(N, page) + 3
    slots = torch.randperm(pool * page, generator=g, device=DEV)[:N].to(torch.int32)
    positions = torch.randint(0, c["ctx"], (N,), generator=g, device=DEV).to(torch.int32)
    slots[N - N // 9:] = NO_SLOT  # the padding of a captured step
    bias = [torch.randn(n * D, generator=g, device=DEV) * 0.3 for n in (heads, kvh, kvh)] if c["bias"] else None
    k, v = (torch.randn(pool, page, kvh, D, generator=g, device=DEV).to(dt) for _ in range(2))
    freqs, scale = _rot_freqs(c)
    return dict(x=x, slots=slots, positions=positions, bias=bias, k=k, v=v, freqs=freqs.to(DEV), scale=scale,
                q=torch.zeros(N, heads * D, dtype=dt, device=DEV))


def _prepare_attn(c, g):
    old, new = _lens(c)
    D, kvh, page, dt = c["dim"], c["kv_heads"], c["page"], TYPES[c["dtype"]]
    heads, N = kvh * c["hpk"], sum(new)
    lens = [o + n for o, n in zip(old, new)]
    tables, _, pool = _layout(g, lens, page, 7)
    # scores of standard deviation 1, some query heads three times as sharp
    q = torch.randn(N, heads, D, generator=g, device=DEV)
    q[:, ::3] *= 3.0
    k, v = (torch.randn(pool, page, kvh, D, generator=g, device=DEV).to(dt) for _ in range(2))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(q=q.to(dt).reshape(N, heads * D), k=k, v=v, tables=tables, lens=_i32(lens), starts=_i32(starts), old=_i32(old),
                new=_i32(new), max_len=max(lens), max_new=max(new), rows=N,
                out=torch.zeros(N, heads * D, dtype=dt, device=DEV))


# ---------------------------------------------------------------------- run
def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn}[state["c"]["kind"]](state)


def _plain_plan(e):
    page, rows = e["c"]["page"], e["rows"]
    old, new = e["old"].long(), e["new"].long()
    B = old.numel()
    ended = new < 0
    fresh = torch.where(ended, 0, new)
    held = (old + page - 1) // page
    lens = torch.where(ended, 0, old + fresh)
    back = torch.where(ended, held, 0)
    take = torch.where(ended, 0, (lens + page - 1) // page - held)
    # pages of ended requests go on top of the free ones, in request order
    b = torch.repeat_interleave(torch.arange(B, device=DEV), back)
    i = torch.arange(b.numel(), device=DEV) - (back.cumsum(0) - back)[b]
    count = e["count"].long()
    stack = e["stack"]
    stack[count + torch.arange(b.numel(), device=DEV)] = e["tables"][b, i]
    # new pages come from the top, in request order
    top = count + b.numel()
    b = torch.repeat_interleave(torch.arange(B, device=DEV), take)
    n = torch.arange(b.numel(), device=DEV)
    e["tables"][b, held[b] + n - (take.cumsum(0) - take)[b]] = stack[top - 1 - n]
    # the step's rows
    ends = fresh.cumsum(0)
    b = torch.repeat_interleave(torch.arange(B, device=DEV), fresh)
    n = torch.arange(b.numel(), device=DEV)
    pos = old[b] + n - (ends - fresh)[b]
    positions = torch.zeros(rows, dtype=torch.int32, device=DEV)
    slots = torch.full((rows,), NO_SLOT, dtype=torch.int32, device=DEV)
    positions[: n.numel()] = pos.int()
    slots[: n.numel()] = e["tables"][b, pos // page] * page + (pos % page).int()
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    taken = take.sum()
    status = torch.stack([taken * 0, taken * 0, ends[-1], taken]).int()
    return dict(tables=e["tables"], lens=lens.int(), starts=starts, positions=positions, slots=slots, stack=stack,
                count=(top - taken).int(), status=status)


def _plain_rope(e):
    c = e["c"]
    N, D, kvh, heads, rot = c["tokens"], c["dim"], c["kv_heads"], c["kv_heads"] * c["hpk"], c["rot"]
    x = e["x"].float()
    if e["bias"]:
        x = x + torch.cat(e["bias"])
    x = x.reshape(N, heads + 2 * kvh, D)
    turn, v = x[:, : heads + kvh], x[:, heads + kvh:]
    angle = e["positions"].double()[:, None] * e["freqs"]
    cos, sin = ((t * e["scale"]).float()[:, None, :] for t in (angle.cos(), angle.sin()))
    a, b = (turn[..., : rot // 2], turn[..., rot // 2: rot]) if c["half"] else (turn[..., 0:rot:2], turn[..., 1:rot:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    both = torch.cat([a, b], -1) if c["half"] else torch.stack([a, b], -1).flatten(-2)
    turn = torch.cat([both, turn[..., rot:]], -1).to(e["q"].dtype)
    used = (e["slots"] >= 0).nonzero()[:, 0]
    at = e["slots"][used].long()
    e["q"][used] = turn[used, :heads].reshape(used.numel(), heads * D)
    e["k"].view(-1, kvh, D)[at] = turn[used, heads:]
    e["v"].view(-1, kvh, D)[at] = v[used].to(e["v"].dtype)
    return dict(q=e["q"], k=e["k"], v=e["v"])


def _plain_attn(e):
    c = e["c"]
    D, kvh, hpk, page = c["dim"], c["kv_heads"], c["hpk"], c["page"]
    B, L, M, N = c["requests"], e["max_len"], e["max_new"], e["rows"]
    # every request's keys and values, padded to the longest
    j = torch.arange(L, device=DEV)
    at = e["tables"].long()[:, j // page] * page + j % page
    k = e["k"].view(-1, kvh, D)[at].float().permute(0, 2, 3, 1).contiguous()
    v = e["v"].view(-1, kvh, D)[at].float().permute(0, 2, 1, 3).contiguous()
    # every request's queries, padded to the most
    i = torch.arange(M, device=DEV)
    row = (e["starts"][:-1].long()[:, None] + i).clamp(max=N - 1)
    q = e["q"].float().view(N, kvh, hpk, D)[row] * D ** -0.5
    q = q.permute(0, 2, 3, 1, 4).reshape(B, kvh, hpk * M, D).contiguous()
    s = torch.matmul(q, k).view(B, kvh, hpk, M, L)
    pos = (e["old"].long()[:, None] + i)[:, :, None]
    seen = j <= pos
    if c["window"]:
        seen = seen & ((pos - j < c["window"]) | (j < c["sinks"]))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, kvh, hpk * M, L), v).view(B, kvh, hpk, M, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, M, kvh * hpk * D)
    return o[i < e["new"][:, None]].to(e["out"].dtype)


# ------------------------------------------------------- the framework's calls
def _descriptors(e):
    import arcllm_amd as arc

    c, p = e["c"], torch.Tensor.data_ptr
    types = {"f16": arc.F16, "bf16": arc.BF16, "f32": arc.F32}
    if c["kind"] == "plan":
        return dict(batch=arc.PagedBatch(requests=c["requests"], tokens=e["rows"], max_pages=e["tables"].shape[1],
                                         max_new=e["max_new"], tables=p(e["tables"]), lens=p(e["lens"]),
                                         starts=p(e["starts"]), positions=p(e["positions"]), slots=p(e["slots"])))
    pages = arc.KvPages(k=p(e["k"]), v=p(e["v"]), num_pages=e["k"].shape[0], page_size=c["page"], kv_heads=c["kv_heads"],
                        head_dim=c["dim"], dtype=types[c["dtype"]])
    if c["kind"] == "rope":
        scaling = dict(plain={}, linear=dict(scaling=arc.ROPE_LINEAR, factor=8.0),
                       yarn=dict(scaling=arc.ROPE_YARN, factor=16.0, original_ctx=8192),
                       factors=dict(freq_factors=_factors(c).numpy()))[c["scaling"]]
        phases, scale = arc.rope_phases(c["rot"], THETA, **scaling)
        phases = torch.from_numpy(phases.view("int64")).to(DEV)
        rope = arc.Rope(rot_dim=c["rot"], layout=arc.ROPE_HALF if c["half"] else arc.ROPE_INTERLEAVED, scale=scale,
                        phases=p(phases))
        batch = arc.PagedBatch(requests=0, tokens=c["tokens"], positions=p(e["positions"]), slots=p(e["slots"]))
        return dict(pages=pages, rope=rope, phases=phases, batch=batch, x=types[c["x"]])
    batch = arc.PagedBatch(requests=c["requests"], tokens=e["rows"], max_pages=e["tables"].shape[1], max_new=e["max_new"],
                           tables=p(e["tables"]), lens=p(e["lens"]), starts=p(e["starts"]))
    space = torch.empty(arc.paged_attention_workspace_bytes(pages, batch, c["hpk"]), dtype=torch.uint8, device=DEV)
    return dict(pages=pages, batch=batch, space=space)


def _run_own(e):
    import arcllm_amd as arc

    c, d, p = e["c"], e["own"], torch.Tensor.data_ptr
    if c["kind"] == "plan":
        arc.paged_plan(d["batch"], p(e["old"]), p(e["new"]), c["page"], p(e["stack"]), e["stack"].numel(), p(e["count"]),
                       p(e["count_out"]), p(e["status"]))
        return dict(tables=e["tables"], lens=e["lens"], starts=e["starts"], positions=e["positions"], slots=e["slots"],
                    stack=e["stack"], count=e["count_out"], status=e["status"])
    if c["kind"] == "rope":
        bias = [p(t) for t in e["bias"]] if e["bias"] else [None, None, None]
        arc.rope_append(d["pages"], d["batch"], d["rope"], d["x"], p(e["x"]), e["x"].shape[1], c["hpk"], p(e["q"]),
                        e["q"].shape[1], q_bias=bias[0], k_bias=bias[1], v_bias=bias[2])
        return dict(q=e["q"], k=e["k"], v=e["v"])
    width = e["q"].shape[1]
    arc.paged_attention(d["pages"], d["batch"], p(e["q"]), width, c["hpk"], p(e["out"]), width, p(d["space"]),
                        window=c["window"], sinks=c["sinks"])
    return e["out"]


# --------------------------------------------------------------------- work
def _seen(c, old, new):
    """(pairs of a query token and a position that it sees, positions seen by any of the
    request's query tokens)."""
    pairs, W, S = 0, c["window"], c["sinks"]
    for pos in range(old, old + new):
        n = pos + 1
        pairs += n if not W or n <= W + S else W + S
    n = old + new
    low = max(0, old + 1 - W) if W else 0  # the first position in the first query's window
    return pairs, n - max(0, low - S)


def work(case):
    c = case
    if c["kind"] == "plan":
        old, new = _lens(c)
        tokens = sum(max(n, 0) for n in new)
        pages = sum(_pages(o, c["page"]) if n == RELEASE else _pages(o + n, c["page"]) - _pages(o, c["page"])
                    for o, n in zip(old, new))
        return dict(bytes=4 * (4 * len(old) + 2 * pages + 2 * (tokens + tokens // 16 + 3) + 6), flops=4 * tokens)
    D, kvh, heads = c["dim"], c["kv_heads"], c["kv_heads"] * c["hpk"]
    if c["kind"] == "rope":
        N = c["tokens"] - c["tokens"] // 9
        cols = (heads + 2 * kvh) * D
        size = 4 if c["x"] == "f32" else 2
        return dict(bytes=N * (cols * (size + 2) + 4) + 4 * c["tokens"] + 4 * cols * c["bias"] + 8 * (c["rot"] // 2),
                    flops=N * ((heads + kvh) * c["rot"] * 3 + cols * c["bias"]))
    old, new = _lens(c)
    pairs, keys = (sum(t) for t in zip(*(_seen(c, o, n) for o, n in zip(old, new))))
    return dict(bytes=2 * (2 * keys * kvh * D + 2 * sum(new) * heads * D) + 4 * _pages(keys, c["page"]),
                flops=4 * pairs * heads * D)


# -------------------------------------------------------------------- exact
def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None  # whole numbers
    e = prepare(c, seed)
    return _exact_rope(c, e) if c["kind"] == "rope" else _exact_attn(c, e)


def _exact_rope(c, e):
    D, kvh, heads, rot = c["dim"], c["kv_heads"], c["kv_heads"] * c["hpk"], c["rot"]
    q, k, v = e["q"].double(), e["k"].double(), e["v"].double()
    used = e["slots"] >= 0
    at, x = e["slots"][used].long(), e["x"][used].double()
    if e["bias"]:
        x = x + torch.cat([t.double() for t in e["bias"]])
    x = x.view(-1, heads + 2 * kvh, D)
    # each pair as a complex number, turned by the position's angle
    first = torch.arange(rot // 2, device=DEV) * (1 if c["half"] else 2)
    second = first + (rot // 2 if c["half"] else 1)
    angle = e["positions"][used].double()[:, None] * e["freqs"][None, :]
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, e["scale"]), angle)[:, None, :]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    q[used] = y[:, :heads].reshape(-1, heads * D)
    k.view(-1, kvh, D)[at] = y[:, heads: heads + kvh]
    v.view(-1, kvh, D)[at] = x[:, heads + kvh:]
    return dict(q=q, k=k, v=v)


def _exact_attn(c, e):
    D, kvh, hpk, page = c["dim"], c["kv_heads"], c["hpk"], c["page"]
    old, new = _lens(c)
    out, first = torch.zeros(e["rows"], kvh, hpk, D, dtype=torch.float64, device=DEV), 0
    q = e["q"].view(-1, kvh, hpk, D)
    for b, (o, n) in enumerate(zip(old, new)):
        held = e["tables"][b, : _pages(o + n, page)].long()
        for g in range(kvh):
            K = e["k"][held, :, g].reshape(-1, D)[: o + n].double()
            V = e["v"][held, :, g].reshape(-1, D)[: o + n].double()
            key = torch.arange(o + n, device=DEV)
            for at in range(0, n, 1024):  # a bound on memory
                m = min(1024, n - at)
                pos = torch.arange(o + at, o + at + m, device=DEV)[:, None]
                hidden = key[None, :] > pos
                if c["window"]:
                    hidden = hidden | ((key[None, :] <= pos - c["window"]) & (key[None, :] >= c["sinks"]))
                bar = torch.zeros(hidden.shape, dtype=torch.float64, device=DEV).masked_fill(hidden, -math.inf)
                for h in range(hpk):
                    s = q[first + at: first + at + m, g, h].double() @ K.t() / math.sqrt(D) + bar
                    out[first + at: first + at + m, g, h] = torch.softmax(s, -1) @ V
        first += n
    return out.view(e["rows"], kvh * hpk * D)
