"""The operators of a serving step that verifies trees of drafted tokens, as a program that
drafts for several requests calls them: the trees' masks and positions from parent
indices, attention of the tree's tokens over a paged KV cache, the walk down the tree
with the accepted rows' move in every layer's cache; and the step's projections in 8-bit
floating point (e4m3) with a scale for each block of 128: the rows' quantisation, the
product, and the gate/up pair with its activation.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what the program holds, ``run(state)`` is one pass,
``exact(case, seed)`` the outputs from the definition in float64.  With ``own`` false a
pass is elementary torch operations in 32 bits; with ``own`` true it is the calls of
``arcllm_amd``.

Request lengths belong to the case; tree shapes, values and page orders come from the seed.  Widths and heads are the 7B shape of the benchmark (hidden 3584, 28 query and 4 kv
heads of 128, feed-forward 18944, vocabulary 152064, 28 layers) and generic ones.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
BLOCK = 128
NONE = -1  # 0xffffffff as int32: no parent, no token


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token's hidden state before its projection: latency
        dict(name="quantize 1 x 3584", kind="quant", rows=1, cols=3584, x="f32"),
        # a long prompt's feed-forward activations before the down projection
        dict(name="quantize 4096 x 18944", kind="quant", rows=4096, cols=18944, x="bf16"),
        # q|k|v of one token: the weights are read once, latency beside it
        dict(name="product 1 x 4608 x 3584", kind="product", rows=1, n=4608, k=3584, gated=0, residual=0, y="f32"),
        # the down projection of a few requests' drafted tokens, added to the residual stream
        dict(name="product 45 x 3584 x 18944", kind="product", rows=45, n=3584, k=18944, gated=0, residual=1, y="f32"),
        # gate and up projection of a long prompt, with the activation
        dict(name="gate/up 4096 x 18944 x 3584", kind="product", rows=4096, n=18944, k=3584, gated=1, residual=0, y="bf16"),
        # the tree of one request
        dict(name="plan 1 x 26", kind="plan", requests=1, nodes=26, chunks=0, chunk=0, ctx=501, words=1),
        # a large server's step: trees, decoding requests and prompts
        dict(name="plan 500 x <=60 mixed", kind="plan", requests=500, nodes=60, chunks=12, chunk=400, ctx=9000, words=2),
        # one request's tree over a short odd context: latency
        dict(name="tree 1 x 26 @ 501", kind="attn", requests=1, nodes=26, chunks=0, chunk=0, ctx=501, words=1, kv_heads=4,
             hpk=7, dim=128, dtype="f16", page=16, window=0, sinks=0),
        # many requests' trees over contexts of all lengths
        dict(name="tree 48 x <=60 @ <=8000", kind="attn", requests=48, nodes=60, chunks=0, chunk=0, ctx=8000, words=2,
             kv_heads=4, hpk=7, dim=128, dtype="f16", page=16, window=0, sinks=0),
        # wide trees in a long-context layer with a window and sinks, beside a prompt's chunk
        dict(name="tree 6 x <=250 + 512 windowed", kind="attn", requests=7, nodes=250, chunks=1, chunk=512, ctx=24000, words=8,
             kv_heads=8, hpk=4, dim=128, dtype="bf16", page=32, window=4096, sinks=4),
        # one request accepts a few drafted tokens: latency
        dict(name="commit 1 x 26", kind="commit", requests=1, nodes=26, chunks=0, chunk=0, ctx=501, words=1, kv_heads=4,
             dim=128, dtype="f16", page=16, layers=28, vocab=152064, logits=""),
        # a step of several requests, from the logits of the target model
        dict(name="commit 24 x <=40 logits", kind="commit", requests=24, nodes=40, chunks=0, chunk=0, ctx=400, words=2,
             kv_heads=4, dim=128, dtype="f16", page=16, layers=28, vocab=152064, logits="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "product", "product", "product", "plan", "attn", "attn", "attn", "commit"])
    if kind == "quant":
        cols = 16 * _log(rng, 1, 1184)
        return dict(kind="quant", rows=_log(rng, 1, min(16000, 4096 * 18944 // cols)), cols=cols,
                    x=rng.choice(["f32", "f16", "bf16"]))
    if kind == "product":
        gated = int(rng.random() < 0.3)
        n, k = _log(rng, 30, 19000), 16 * _log(rng, 3, 1184)
        most = int(4096 * 18944 * 3584 * 0.9 / n / k * (2 - gated))
        y = rng.choice(["f32", "f16", "bf16"])
        return dict(kind="product", rows=_log(rng, 1, max(2, min(4096, most))), n=n, k=k, gated=gated,
                    residual=int(not gated and rng.random() < 0.5), y=y)
    nodes = _log(rng, 2, 250)
    words = (nodes + 31) // 32 + rng.randint(0, 1)
    more = dict(nodes=nodes, words=words)
    heads = dict(kv_heads=rng.choice([1, 2, 3, 4, 5, 8]), dim=rng.choice([64, 128, 128]), dtype=rng.choice(["f16", "bf16"]),
                 page=rng.choice([8, 16, 16, 32, 64]))
    if kind == "plan":
        B = _log(rng, 1, min(700, 40000 // nodes))
        return dict(kind="plan", requests=B, chunks=rng.randint(0, B // 20), chunk=32 * words + _log(rng, 1, 500),
                    ctx=_log(rng, 2, 30000), **more)
    if kind == "commit":
        B, logits = _log(rng, 1, 40), rng.choice(["", "f32", "f16", "bf16"])
        while B > 1 and B * nodes > 1500:
            B -= 1
        return dict(kind="commit", requests=B, chunks=rng.randint(0, 1) if B > 2 and not logits else 0,
                    chunk=32 * words + _log(rng, 1, 100), ctx=_log(rng, 2, 400), layers=rng.randint(1, 28),
                    vocab=_log(rng, 1000, 130000), logits=logits, **heads, **more)
    hpk = rng.randint(1, 8)
    B = _log(rng, 1, 64)
    ctx = _log(rng, 2, 30000)
    chunks = 1 if B > 1 and rng.random() < 0.3 else 0
    chunk = 32 * words + _log(rng, 1, 200)
    each = (chunk if chunks else nodes) * heads["kv_heads"] * hpk
    while B > 2 and B * each * ctx > 3e8:
        B -= 1
    while B * each * ctx > 3e8:
        ctx = ctx * 2 // 3
    window = rng.choice([0, 0, _log(rng, 8, 4096)])
    return dict(kind="attn", requests=B, chunks=chunks, chunk=chunk, ctx=ctx, hpk=hpk, window=window,
                sinks=rng.randint(0, 8) if window else 0, **heads, **more)


# --------------------------------------------------------- lengths and trees
def _shape(c, seed=0):
    """For every request: positions held before the step, its rows' parents in a tree (None
    for a prompt's chunk) and the number of its rows."""
    rng = random.Random("%s %s %s %s" % (c["requests"], c["nodes"], c["ctx"], c["chunks"]))
    grow = random.Random(int(seed))
    B, shapes = c["requests"], []
    chunks = set(rng.sample(range(B), c["chunks"]))
    for b in range(B):
        held = c["ctx"] if b == 0 else _log(rng, max(1, c["ctx"] // 40), c["ctx"])
        if b in chunks:
            shapes.append((held, None, c["chunk"] if b == 0 else rng.randint(32 * c["words"] + 1, c["chunk"])))
            continue
        n = c["nodes"] if b == 0 else rng.randint((c["nodes"] + 1) // 2, c["nodes"])
        if rng.random() < 0.1:
            n = 1  # nothing drafted: a plain decode step
        # node 0 is the last token, each other node continues one of those before it
        parents = [NONE] + [grow.randint((i - 1) // 3, i - 1) for i in range(1, n)]
        shapes.append((held, parents, n))
    return shapes


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p == NONE else d[p] + 1)
    return d


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------- inputs
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + stream * 7919 + 4242) & 0x7FFFFFFFFFFF)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _blocks(n):
    return -(-n // BLOCK)


def _spread(t, rows, cols):
    """Values of a matrix's blocks (1 or 128 rows by 128 columns) for each of its elements."""
    t = t.repeat_interleave(BLOCK, 1)[:, :cols]
    return t if t.shape[0] == rows else t.repeat_interleave(BLOCK, 0)[:rows]


def _scale_of(most):
    """The scale of a block from its largest magnitude: that becomes 448, e4m3's largest."""
    s = (most / 448.0).clamp(min=2.0 ** -126)
    return torch.where(torch.isfinite(most), s, math.nan)


def _quantize_rows(x):
    """(e4m3 values, scales [blocks][rows]) of the rows of x, 32 bits."""
    M, K = x.shape
    most = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(M, -1, BLOCK).abs().amax(-1)
    s = _scale_of(most)
    return (x / _spread(s, M, K)).to(E4M3), s.t().contiguous()


def _weights(g, n, k):
    """(e4m3 values [n][k], scales [blocks of n][blocks of k]) of normal weights."""
    w = torch.randn(n, k, generator=g, device=DEV) * 0.03
    most = torch.nn.functional.pad(w.abs(), (0, -k % BLOCK, 0, -n % BLOCK)).view(_blocks(n), BLOCK, _blocks(k), BLOCK)
    s = _scale_of(most.amax((1, 3)))
    return (w / _spread(s, n, k)).to(E4M3), s


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    c, g = case, _gen(seed, 0)
    if c["kind"] == "quant":
        e = _prepare_quant(c, g)
    elif c["kind"] == "product":
        e = _prepare_product(c, g)
    else:
        e = _prepare_tree(c, g, seed)
    e["c"] = c
    if own:  # the descriptors and workspace that a program of the framework keeps
        e["own"] = _descriptors(e)
    return e


def _activations(g, rows, cols):
    """Rows of different size with a few channels far above the others."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.rand(rows, 1, generator=g, device=DEV) * 3 + 0.1
    x[:, ::97] *= 12.0
    return x


def _prepare_quant(c, g):
    M, K = c["rows"], c["cols"]
    return dict(x=_activations(g, M, K).to(TYPES[c["x"]]), q=torch.zeros(M, K, dtype=E4M3, device=DEV),
                scales=torch.zeros(_blocks(K), M, device=DEV))


def _prepare_product(c, g):
    M, N, K = c["rows"], c["n"], c["k"]
    x, xs = _quantize_rows(_activations(g, M, K))
    e = dict(x=x, xs=xs, y=torch.zeros(M, N, dtype=TYPES[c["y"]], device=DEV), w=[_weights(g, N, K)])
    if c["gated"]:
        e["w"].append(_weights(g, N, K))
    if c["residual"]:
        e["res"] = (torch.randn(M, N, generator=g, device=DEV) * 4.0).to(TYPES[c["y"]])
    return e


def _prepare_tree(c, g, seed):
    shapes = _shape(c, seed)
    B, words, page = c["requests"], c["words"], c.get("page", 16)
    held, rows = [s[0] for s in shapes], [s[2] for s in shapes]
    N = sum(rows)
    parents, depths = [], []
    for _, tree, n in shapes:
        parents += tree if tree is not None else [NONE] + list(range(n - 1))
        depths += _depths(tree) if tree is not None else list(range(n))
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    lens = [o + n for o, n in zip(held, rows)]
    spare = N // 16 + 3  # a step's buffers hold some more rows than it uses
    e = dict(held=_i32(held), new=_i32(rows), lens=_i32(lens), starts=_i32(starts), parents=_i32(parents + [NONE] * spare),
             rows=N, buffer=N + spare, max_len=max(lens), max_new=max(rows),
             deepest=max(max(_depths(t)) for _, t, _ in shapes if t is not None) if c["chunks"] < B else 0,
             positions=torch.zeros(N + spare, dtype=torch.int32, device=DEV),
             masks=torch.zeros(N + spare, words, dtype=torch.int32, device=DEV))
    if c["kind"] == "plan":
        return e
    # pages of every request in a random order over the pool, free ones behind
    need = [_pages(n, page) for n in lens]
    total, longest = sum(need), max(need)
    order = torch.randperm(total + 7, generator=g, device=DEV).to(torch.int32)
    need = torch.tensor(need, device=DEV)
    col = torch.arange(longest, device=DEV)[None, :]
    at = (need.cumsum(0) - need)[:, None] + col
    e["tables"] = torch.where(col < need[:, None], order[at.clamp(max=total - 1).long()], 0).to(torch.int32).contiguous()
    pool, kvh, D, dt = total + 7, c["kv_heads"], c["dim"], TYPES[c["dtype"]]
    if c["kind"] == "attn":
        e["positions"][:N] = e["held"].long().repeat_interleave(e["new"].long()).int() + _i32(depths)
        e["masks"][:N] = _masks(e, c)
        heads = kvh * c["hpk"]
        # scores of standard deviation 1, some query heads three times as sharp
        q = torch.randn(N, heads, D, generator=g, device=DEV)
        q[:, ::3] *= 3.0
        e["q"] = q.to(dt).view(N, heads * D)
        e["k"], e["v"] = (torch.randn(pool, page, kvh, D, generator=g, device=DEV).to(dt) for _ in range(2))
        e["out"] = torch.zeros(N, heads * D, dtype=dt, device=DEV)
        return e
    e["k"], e["v"] = (torch.randn(c["layers"], pool, page, kvh, D, generator=g, device=DEV, dtype=dt) for _ in range(2))
    # the target's token after each row; two of three drafted tokens are what it says after their parents
    target = torch.randint(0, c["vocab"], (N,), generator=g, device=DEV)
    first = e["starts"][:-1].long().repeat_interleave(e["new"].long())
    said = target[first + e["parents"][:N].long().clamp(min=0)]
    other = torch.randint(0, c["vocab"], (N,), generator=g, device=DEV)
    e["drafts"] = torch.where(torch.rand(N, generator=g, device=DEV) < 0.67, said, other).int()
    if c["logits"]:
        logits = torch.randn(N, c["vocab"], generator=g, device=DEV)
        logits.scatter_(1, target[:, None], 8.0)
        e["logits"] = logits.to(TYPES[c["logits"]])
        e["targets"] = torch.zeros(N, dtype=torch.int32, device=DEV)
    else:
        e["targets"] = target.int()
    e["stack"] = torch.zeros(pool, dtype=torch.int32, device=DEV)
    e["stack"][:7] = order[total:]
    full = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    e.update(count=_i32([7]), count_out=full(1), lens_out=full(B), counts=full(B), tokens=full(N))
    return e


# ---------------------------------------------------------------------- run
def run(state):
    if own:
        return _run_own(state)
    return {"quant": _plain_quant, "product": _plain_product, "plan": _plain_plan, "attn": _plain_attn,
            "commit": _plain_commit}[state["c"]["kind"]](state)


def _plain_quant(e):
    q, s = _quantize_rows(e["x"].float())
    return dict(q=q, scales=s)


def _plain_product(e):
    M, K = e["x"].shape
    x = e["x"].float() * _spread(e["xs"].t(), M, K)
    ys = [x @ (w.float() * _spread(s, w.shape[0], K)).t() for w, s in e["w"]]
    y = ys[0] / (1 + (-ys[0]).exp()) * ys[1] if e["c"]["gated"] else ys[0]
    if e["c"]["residual"]:
        y = y + e["res"].float()
    return y.to(e["y"].dtype)


def _row_places(e):
    """Each row's request and its index in the request."""
    b = torch.repeat_interleave(torch.arange(e["new"].numel(), device=DEV), e["new"].long(), output_size=e["rows"])
    return b, torch.arange(e["rows"], device=DEV) - e["starts"].long()[b]


def _masks(e, c):
    """Bits of the nodes from which each row of a tree descends, its own among them."""
    b, i = _row_places(e)
    first = e["starts"].long()[b]
    parents = e["parents"][: e["rows"]].long()
    tree = (e["new"].long() <= 32 * c["words"])[b]
    bits = torch.zeros(e["rows"], 32 * c["words"] + 1, dtype=torch.int64, device=DEV)
    at = torch.where(tree, i, NONE)
    for _ in range(e["deepest"] + 1):  # one generation further up each time; rows that are done write the last column
        bits.scatter_(1, torch.where(at >= 0, at, 32 * c["words"])[:, None], 1)
        at = torch.where(at >= 0, parents[first + at.clamp(min=0)], NONE)
    words = (bits[:, :-1].view(e["rows"], -1, 32) << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def _plain_plan(e):
    c, N = e["c"], e["rows"]
    b, i = _row_places(e)
    masks = _masks(e, c)
    ones = ((masks.long()[:, :, None] >> torch.arange(32, device=DEV)) & 1).sum((1, 2))
    depth = torch.where((e["new"].long() <= 32 * c["words"])[b], ones - 1, i)
    e["masks"][:N] = masks
    e["positions"][:N] = (e["lens"].long() - e["new"].long())[b].int() + depth.int()
    return dict(masks=e["masks"], positions=e["positions"])


def _plain_attn(e):
    c = e["c"]
    D, kvh, hpk, page, words = c["dim"], c["kv_heads"], c["hpk"], c["page"], c["words"]
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
    # the context, and of the step's own rows those that the mask names (a chunk: those up to it)
    base = (e["lens"] - e["new"]).long()[:, None]
    rel = j - base
    at = rel.clamp(0, 32 * words - 1)
    bits = e["masks"][:N].long()[row].gather(2, (at // 32)[:, None, :].expand(B, M, L))
    named = ((bits >> (at % 32)[:, None, :]) & 1).bool()
    chunk = (e["new"].long() > 32 * words)[:, None, None]
    named = torch.where(chunk, rel[:, None, :] <= i[:, None], named & (rel < 32 * words)[:, None, :])
    seen = (rel < 0)[:, None, :] | named
    if c["window"]:
        pos = e["positions"].long()
        place = torch.where(rel < 0, j, pos[(e["starts"][:-1].long()[:, None] + rel).clamp(0, N - 1)])[:, None, :]
        seen = seen & ((pos[row][:, :, None] - place < c["window"]) | (place < c["sinks"]))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, kvh, hpk * M, L), v).view(B, kvh, hpk, M, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, M, kvh * hpk * D)
    return o[i < e["new"][:, None]].to(e["out"].dtype)


def _plain_commit(e):
    c, N = e["c"], e["rows"]
    B, T, page = c["requests"], e["max_new"], c["page"]
    target = e["targets"].long()
    if c["logits"]:  # the largest, the lowest of equals
        x = e["logits"]
        target = torch.where(x == x.amax(-1, keepdim=True), torch.arange(c["vocab"], device=DEV), c["vocab"]).amin(-1)
    starts, new = e["starts"][:-1].long(), e["new"].long()
    i = torch.arange(T, device=DEV)
    row = (starts[:, None] + i).clamp(max=N - 1)
    there = i < new[:, None]
    parents = torch.where(there, e["parents"].long()[row], NONE - 1)
    drafts, said = e["drafts"].long()[row], target[row]
    chunk = new > 32 * c["words"]
    # down the tree: the first child that holds the target's token
    node, alive = torch.zeros(B, dtype=torch.int64, device=DEV), ~chunk
    path = torch.full((B, T + 1), T, dtype=torch.int64, device=DEV)
    path[:, 0] = 0
    for step in range(1, e["deepest"] + 1):
        want = said.gather(1, node[:, None])
        fits = (parents == node[:, None]) & (drafts == want) & alive[:, None]
        next_ = torch.where(fits, i, T).amin(1)
        alive = alive & (next_ < T)
        node = torch.where(alive, next_, node)
        path[:, step] = torch.where(alive, next_, T)
    kept = torch.where(chunk, 1, (path < T).sum(1))
    path[:, 0] = torch.where(chunk, new - 1, 0)
    length = torch.where(chunk, new, kept)
    lens = e["lens"].long() - new + length
    # the tokens that each request goes on with
    tokens = torch.full((N,), NONE, dtype=torch.int32, device=DEV)
    b = torch.repeat_interleave(torch.arange(B, device=DEV), kept)
    n = torch.arange(b.numel(), device=DEV) - (kept.cumsum(0) - kept)[b]
    from_ = path[b, n]
    tokens[starts[b] + n] = said[b, from_].int()
    # the accepted rows' keys and values to the places behind the context, in every layer
    moves = ~chunk[b]
    b, n, from_ = b[moves], n[moves], from_[moves]
    base = (e["lens"].long() - new)[b]
    slot = lambda pos: e["tables"].long()[b, pos // page] * page + pos % page  # noqa: E731
    to, of = slot(base + n), slot(base + from_)
    flat = (c["layers"], -1, c["kv_heads"], c["dim"])
    e["k"].view(flat)[:, to] = e["k"].view(flat)[:, of]
    e["v"].view(flat)[:, to] = e["v"].view(flat)[:, of]
    # pages that held rejected rows only go back, in request order
    low, high = (lens + page - 1) // page, (e["lens"].long() + page - 1) // page
    back = high - low
    b = torch.repeat_interleave(torch.arange(B, device=DEV), back)
    n = torch.arange(b.numel(), device=DEV)
    e["stack"][e["count"].long() + n] = e["tables"][b, low[b] + n - (back.cumsum(0) - back)[b]]
    return dict(counts=kept.int(), tokens=tokens, targets=target.int(), lens=lens.int(), k=e["k"], v=e["v"],
                stack=e["stack"], count=(e["count"].long() + back.sum()).int())


# ------------------------------------------------------- the framework's calls
def _descriptors(e):
    import arcllm_amd as arc

    c, p = e["c"], torch.Tensor.data_ptr
    types = {"f16": arc.F16, "bf16": arc.BF16, "f32": arc.F32}
    if c["kind"] == "quant":
        return dict(rows=arc.Fp8Rows(q=p(e["q"]), scales=p(e["scales"]), rows=c["rows"], cols=c["cols"]), x=types[c["x"]])
    if c["kind"] == "product":
        weights = [arc.Fp8Weights(w=p(w), scales=p(s), rows=c["n"], cols=c["k"]) for w, s in e["w"]]
        rows = arc.Fp8Rows(q=p(e["x"]), scales=p(e["xs"]), rows=c["rows"], cols=c["k"])
        size = arc.fp8_gemm_workspace_bytes(c["n"], c["k"], c["rows"], gated=bool(c["gated"]))
        return dict(weights=weights, rows=rows, y=types[c["y"]], space=torch.empty(size, dtype=torch.uint8, device=DEV))
    tables = e.get("tables")
    batch = arc.PagedBatch(requests=c["requests"], tokens=e["buffer"] if c["kind"] == "plan" else e["rows"],
                           max_pages=0 if tables is None else tables.shape[1], max_new=e["max_new"],
                           tables=None if tables is None else p(tables), lens=p(e["lens"]), starts=p(e["starts"]),
                           positions=p(e["positions"]))
    tree = arc.Tree(parents=p(e["parents"]), masks=p(e["masks"]), mask_words=c["words"])
    if c["kind"] == "plan":
        return dict(batch=batch, tree=tree)
    layers = [(e["k"], e["v"])] if c["kind"] == "attn" else list(zip(e["k"], e["v"]))
    pages = [arc.KvPages(k=p(k), v=p(v), num_pages=k.shape[0], page_size=c["page"], kv_heads=c["kv_heads"],
                         head_dim=c["dim"], dtype=types[c["dtype"]]) for k, v in layers]
    if c["kind"] == "attn":
        size = arc.tree_attention_workspace_bytes(pages[0], batch, c["hpk"])
    else:
        size = arc.tree_commit_workspace_bytes(batch)
    return dict(batch=batch, tree=tree, pages=pages, logits=types.get(c.get("logits"), arc.F32),
                space=torch.empty(size, dtype=torch.uint8, device=DEV))


def _run_own(e):
    import arcllm_amd as arc

    c, d, p = e["c"], e["own"], torch.Tensor.data_ptr
    if c["kind"] == "quant":
        arc.fp8_quantize(d["x"], p(e["x"]), c["cols"], d["rows"])
        return dict(q=e["q"], scales=e["scales"])
    if c["kind"] == "product":
        if c["gated"]:
            arc.fp8_gateup(*d["weights"], d["rows"], d["y"], p(e["y"]), c["n"], p(d["space"]))
        else:
            arc.fp8_gemm(d["weights"][0], d["rows"], d["y"], p(e["y"]), c["n"], p(d["space"]),
                         residual=p(e["res"]) if c["residual"] else None, ldr=c["n"])
        return e["y"]
    if c["kind"] == "plan":
        arc.tree_plan(d["batch"], d["tree"])
        return dict(masks=e["masks"], positions=e["positions"])
    if c["kind"] == "attn":
        width = e["q"].shape[1]
        arc.tree_attention(d["pages"][0], d["batch"], d["tree"], p(e["q"]), width, c["hpk"], p(e["out"]), width, p(d["space"]),
                           window=c["window"], sinks=c["sinks"])
        return e["out"]
    arc.tree_commit(d["pages"], d["batch"], d["tree"], p(e["drafts"]), p(e["targets"]), p(e["lens_out"]), p(e["counts"]),
                    p(e["tokens"]), p(d["space"]), free_pages=p(e["stack"]), num_pages=e["stack"].numel(),
                    free_count=p(e["count"]), free_count_out=p(e["count_out"]),
                    logits=p(e["logits"]) if c["logits"] else None, logits_dtype=d["logits"], ldl=c["vocab"], vocab=c["vocab"])
    return dict(counts=e["counts"], tokens=e["tokens"], targets=e["targets"], lens=e["lens_out"], k=e["k"], v=e["v"],
                stack=e["stack"], count=e["count_out"])


# --------------------------------------------------------------------- work
def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "quant":
        M, K = c["rows"], c["cols"]
        return dict(bytes=M * K * (size[c["x"]] + 1) + 4 * M * _blocks(K), flops=3 * M * K)
    if c["kind"] == "product":
        M, N, K, mats = c["rows"], c["n"], c["k"], 1 + c["gated"]
        held = mats * (N * K + 4 * _blocks(N) * _blocks(K)) + M * K + 4 * M * _blocks(K)
        return dict(bytes=held + M * N * size[c["y"]] * (1 + c["residual"]), flops=2 * M * N * K * mats)
    shapes = _shape(c)
    rows, B = sum(s[2] for s in shapes), c["requests"]
    if c["kind"] == "plan":
        trees = sum(n for _, tree, n in shapes if tree is not None)
        return dict(bytes=4 * (2 * B + 1 + trees * (1 + c["words"]) + rows), flops=rows)
    D, kvh = c["dim"], c["kv_heads"]
    if c["kind"] == "commit":
        logits = rows * c["vocab"] * size[c["logits"]] if c["logits"] else 4 * rows
        kept = 2 * sum(tree is not None for _, tree, _ in shapes)  # about two rows of a tree move
        return dict(bytes=logits + 4 * (3 * rows + 6 * B) + 2 * kept * c["layers"] * 2 * kvh * D * 2, flops=rows)
    W, S, pairs, keys = c["window"], c["sinks"], 0, 0
    for held, tree, n in shapes:
        for d in _depths(tree) if tree is not None else range(n):
            pos = held + d
            pairs += pos + 1 if not W or pos + 1 <= W + S else W + S
        low = max(0, held + 1 - W) if W else 0  # the first position in the first row's window
        keys += held + n - max(0, low - S)
    heads = kvh * c["hpk"]
    return dict(bytes=2 * (2 * keys * kvh * D + 2 * rows * heads * D) + 4 * (_pages(keys, c["page"]) + rows * c["words"]),
                flops=4 * pairs * heads * D)


# -------------------------------------------------------------------- exact
def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None  # whole numbers
    e = prepare(c, seed)
    return {"quant": _exact_quant, "product": _exact_product, "attn": _exact_attn, "commit": _exact_commit}[c["kind"]](c, e, seed)


def _exact_quant(c, e, seed):
    """Scales from the definition; the values that the 8 bits stand for, unrounded."""
    M, K = c["rows"], c["cols"]
    scales = torch.zeros(_blocks(K), M, dtype=torch.float64, device=DEV)
    q = torch.zeros(M, K, dtype=torch.float64, device=DEV)
    for n in range(_blocks(K)):
        x = e["x"][:, n * BLOCK: (n + 1) * BLOCK].double()
        scales[n] = torch.maximum(x.max(1).values, -x.min(1).values) / 448
        q[:, n * BLOCK: (n + 1) * BLOCK] = x / scales[n][:, None]
    return dict(q=q, scales=scales)


def _exact_product(c, e, seed):
    M, N, K = c["rows"], c["n"], c["k"]
    ys = [torch.zeros(M, N, dtype=torch.float64, device=DEV) for _ in e["w"]]
    for n in range(_blocks(K)):
        cols = slice(n * BLOCK, (n + 1) * BLOCK)
        x = e["x"][:, cols].double() * e["xs"][n].double()[:, None]
        for y, (w, s) in zip(ys, e["w"]):
            ws = s[:, n].double()[torch.arange(N, device=DEV) // BLOCK]
            y += x @ (w[:, cols].double() * ws[:, None]).t()
    y = ys[0]
    if c["gated"]:
        y = ys[0] * torch.sigmoid(ys[0]) * ys[1]
    return y + e["res"].double() if c["residual"] else y


def _exact_attn(c, e, seed):
    D, kvh, hpk, page = c["dim"], c["kv_heads"], c["hpk"], c["page"]
    out, first = torch.zeros(e["rows"], kvh, hpk, D, dtype=torch.float64, device=DEV), 0
    q = e["q"].view(-1, kvh, hpk, D)
    for b, (held, tree, n) in enumerate(_shape(c, seed)):
        # who sees whom among the step's own rows, from the parents
        sees = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            p = i
            while p != NONE:
                sees[i, p] = True
                p = (tree[p] if p else NONE) if tree is not None else p - 1
        depth = torch.tensor(_depths(tree) if tree is not None else list(range(n)), device=DEV)
        seen = torch.cat([torch.ones(n, held, dtype=torch.bool), sees], 1).to(DEV)
        place = torch.cat([torch.arange(held, device=DEV), held + depth])
        if c["window"]:
            seen &= (held + depth[:, None] - place < c["window"]) | (place < c["sinks"])
        bar = torch.zeros(seen.shape, dtype=torch.float64, device=DEV).masked_fill(~seen, -math.inf)
        pages = e["tables"][b, : _pages(held + n, page)].long()
        for g in range(kvh):
            K = e["k"][pages, :, g].reshape(-1, D)[: held + n].double()
            V = e["v"][pages, :, g].reshape(-1, D)[: held + n].double()
            for h in range(hpk):
                s = q[first: first + n, g, h].double() @ K.t() / math.sqrt(D) + bar
                out[first: first + n, g, h] = torch.softmax(s, -1) @ V
        first += n
    return out.view(e["rows"], kvh * hpk * D)


def _exact_commit(c, e, seed):
    """Keys and values after the walk, a request at a time; whole numbers have no such value."""
    said = (e["logits"].max(1).indices if c["logits"] else e["targets"]).tolist()
    drafts, starts, tables, page = e["drafts"].tolist(), e["starts"].tolist(), e["tables"].tolist(), c["page"]
    to, of = [], []
    for b, (held, tree, n) in enumerate(_shape(c, seed)):
        node, place = 0, 0
        while tree is not None:
            child = [i for i in range(node + 1, n) if tree[i] == node and drafts[starts[b] + i] == said[starts[b] + node]]
            if not child:
                break
            node, place = child[0], place + 1
            for slots, pos in ((to, held + place), (of, held + node)):
                slots.append(tables[b][pos // page] * page + pos % page)
    none = dict.fromkeys(("counts", "tokens", "targets", "lens", "stack", "count"))
    moved = {}
    for name in ("k", "v"):
        t = e[name].double().view(c["layers"], -1, c["kv_heads"] * c["dim"])
        rows = t[:, of]
        t[:, to] = rows
        moved[name] = t.view(e[name].shape)
    return dict(none, **moved)
