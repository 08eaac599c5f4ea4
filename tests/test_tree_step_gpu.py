"""Steps that verify trees of drafted tokens, as a server runs them: plan, masks, per layer 8-bit projections,
rotary positions with the cache write, attention and the feed-forward pair, logits and the commit, which the
next step takes up; eagerly against float64 stage by stage, and captured."""
import numpy as np
import pytest
import torch

import arcllm_amd as arc
import fp8_lib as fl
import paged_lib as pl
import tree_lib as tl

pytestmark = pytest.mark.gpu

SEED = 0x57E9
B, HID, KV, HPK, DIM, FFN, VOCAB, LAYERS, PAGE, POOL, MAX_PAGES = 3, 256, 2, 3, 64, 400, 12, 2, 4, 120, 30
HEADS = KV * HPK
QKV = (HEADS + 2 * KV) * DIM
ROWS = 64  # of the step's buffers
WORDS = 1


class TorchStream:
    def __init__(self):
        self.handle = torch.cuda.current_stream().cuda_stream


def p(t):
    return t.data_ptr()


def i32(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


class Server:
    """The weights and the cache of a small model, and a step's buffers."""

    def __init__(self):
        rng = np.random.default_rng(SEED)
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.layers = []
        for _ in range(LAYERS):
            layer = {}
            for name, n, k in (("qkv", QKV, HID), ("o", HID, HEADS * DIM), ("gate", FFN, HID), ("up", FFN, HID), ("down", HID, FFN)):
                q, s = fl.weights(rng, n, k)
                layer[name] = (q, s * 0.01, cuda(q), cuda(s * np.float32(0.01)))
            layer["bias"] = [cuda(rng.standard_normal(n * DIM).astype(np.float32)) for n in (HEADS, KV, KV)]
            layer["kv"] = [torch.zeros(POOL, PAGE, KV, DIM, dtype=torch.float16, device="cuda") for _ in range(2)]
            self.layers.append(layer)
        q, s = fl.weights(rng, VOCAB, HID)
        self.head = (q, s, cuda(q), cuda(s))
        self.embed = cuda(rng.standard_normal((VOCAB, HID)).astype(np.float32))
        self.phases = torch.from_numpy(arc.rope_phases(DIM, 1e4)[0].view(np.int64)).cuda()
        self.tables, self.lens, self.starts = i32(B, MAX_PAGES), i32(B), i32(B + 1)
        self.positions, self.slots, self.new, self.status = i32(ROWS), i32(ROWS), i32(B), i32(4)
        self.stack, self.count = torch.arange(POOL, dtype=torch.int32, device="cuda"), i32(1, fill=POOL)
        self.parents, self.masks, self.drafts, self.targets = i32(ROWS), i32(ROWS, WORDS), i32(ROWS), i32(ROWS)
        self.counts, self.tokens = i32(B), i32(ROWS)
        f32 = lambda n: torch.zeros(ROWS, n, device="cuda")  # noqa: E731
        self.h, self.x, self.logits, self.qkv = f32(HID), f32(HID), f32(VOCAB), f32(QKV)
        self.q, self.attn = (torch.zeros(ROWS, HEADS * DIM, dtype=torch.float16, device="cuda") for _ in range(2))
        self.act = torch.zeros(ROWS, FFN, dtype=torch.bfloat16, device="cuda")
        self.q8 = torch.zeros(ROWS, 512, dtype=torch.uint8, device="cuda")
        self.s8 = torch.zeros(4, ROWS, device="cuda")
        self.batch = arc.PagedBatch(B, ROWS, MAX_PAGES, ROWS, p(self.tables), p(self.lens), p(self.starts), p(self.positions), p(self.slots))
        self.tree = arc.Tree(p(self.parents), p(self.masks), WORDS)
        self.pages = [arc.KvPages(p(l["kv"][0]), p(l["kv"][1]), POOL, PAGE, KV, DIM) for l in self.layers]
        size = max([arc.fp8_gemm_workspace_bytes(n, k, ROWS) for n, k in ((QKV, HID), (HID, HEADS * DIM), (HID, FFN), (VOCAB, HID))]
                   + [arc.fp8_gemm_workspace_bytes(FFN, HID, ROWS, gated=True), arc.tree_commit_workspace_bytes(self.batch),
                      arc.tree_attention_workspace_bytes(self.pages[0], self.batch, HPK)])
        self.ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")

    def weights(self, w):
        return arc.Fp8Weights(p(w[2]), p(w[3]), *w[0].shape)

    def rows(self, cols):
        return arc.Fp8Rows(p(self.q8), p(self.s8), ROWS, cols, 512, ROWS)

    def norm(self):
        self.x.copy_(self.h * torch.rsqrt((self.h * self.h).mean(1, keepdim=True) + 1e-6))

    # the check of a stage, if any, is called with what went in
    def step(self, check=None):
        st = TorchStream()
        see = check or (lambda *a: None)
        arc.paged_plan(self.batch, p(self.lens), p(self.new), PAGE, p(self.stack), POOL, p(self.count), p(self.count), p(self.status), stream=st)
        arc.tree_plan(self.batch, self.tree, stream=st)
        see("plan")
        self.h.copy_(self.embed[self.drafts.long().clamp(0, VOCAB - 1)])
        for n, l in enumerate(self.layers):
            self.norm()
            arc.fp8_quantize(arc.F32, p(self.x), HID, self.rows(HID), stream=st)
            see("quantize", self.x, HID)
            arc.fp8_gemm(self.weights(l["qkv"]), self.rows(HID), arc.F32, p(self.qkv), QKV, p(self.ws), stream=st)
            see("gemm", l["qkv"], self.qkv, arc.F32, None)
            bias = [p(t) for t in l["bias"]]
            arc.rope_append(self.pages[n], self.batch, arc.Rope(p(self.phases), DIM), arc.F32, p(self.qkv), QKV, HPK, p(self.q), HEADS * DIM,
                            *bias, stream=st)
            arc.tree_attention(self.pages[n], self.batch, self.tree, p(self.q), HEADS * DIM, HPK, p(self.attn), HEADS * DIM, p(self.ws), stream=st)
            see("attention", l)
            arc.fp8_quantize(arc.F16, p(self.attn), HEADS * DIM, self.rows(HEADS * DIM), stream=st)
            see("quantize", self.attn, HEADS * DIM)
            before = None if check is None else self.h.clone()
            arc.fp8_gemm(self.weights(l["o"]), self.rows(HEADS * DIM), arc.F32, p(self.h), HID, p(self.ws), residual=p(self.h), ldr=HID, stream=st)
            see("gemm", l["o"], self.h, arc.F32, before)
            self.norm()
            arc.fp8_quantize(arc.F32, p(self.x), HID, self.rows(HID), stream=st)
            arc.fp8_gateup(self.weights(l["gate"]), self.weights(l["up"]), self.rows(HID), arc.BF16, p(self.act), FFN, p(self.ws), stream=st)
            see("gateup", l, self.act)
            arc.fp8_quantize(arc.BF16, p(self.act), FFN, self.rows(FFN), stream=st)
            see("quantize", self.act, FFN)
            before = None if check is None else self.h.clone()
            arc.fp8_gemm(self.weights(l["down"]), self.rows(FFN), arc.F32, p(self.h), HID, p(self.ws), residual=p(self.h), ldr=HID, stream=st)
            see("gemm", l["down"], self.h, arc.F32, before)
        self.norm()
        arc.fp8_quantize(arc.F32, p(self.x), HID, self.rows(HID), stream=st)
        arc.fp8_gemm(self.weights(self.head), self.rows(HID), arc.F32, p(self.logits), VOCAB, p(self.ws), stream=st)
        see("gemm", self.head, self.logits, arc.F32, None)
        see("before commit")
        arc.tree_commit(self.pages, self.batch, self.tree, p(self.drafts), p(self.targets), p(self.lens), p(self.counts), p(self.tokens),
                        p(self.ws), free_pages=p(self.stack), num_pages=POOL, free_count=p(self.count), free_count_out=p(self.count),
                        logits=p(self.logits), logits_dtype=arc.F32, ldl=VOCAB, vocab=VOCAB, stream=st)

    def draft(self, shapes, tokens):
        """Puts a step's trees (or prompts' chunks) and their tokens in place."""
        new, at = [s if isinstance(s, int) else len(s) for s in shapes], 0
        parents = np.full(ROWS, arc.NO_PARENT, np.uint32)
        for s, n in zip(shapes, new):
            if not isinstance(s, int):
                parents[at: at + n] = s
            at += n
        self.parents.copy_(torch.from_numpy(parents.view(np.int32)))
        self.drafts.copy_(torch.from_numpy(np.pad(np.asarray(tokens, np.int32), (0, ROWS - at))))
        self.new.copy_(torch.tensor(new, dtype=torch.int32))

    STATE = ("tables", "lens", "starts", "positions", "slots", "stack", "count", "counts", "tokens", "targets", "h", "attn", "act", "logits", "masks")


class Check:
    """Each stage against its statement, from what the stage was given."""

    def __init__(self, s):
        self.s, self.seen = s, set()

    def __call__(self, stage, *args):
        torch.cuda.synchronize()
        self.seen.add(stage)
        getattr(self, stage.replace(" ", "_"))(*args)

    def used(self):
        return int(self.s.starts[-1])

    def codes(self, cols):
        return self.s.q8[:, :cols].cpu().numpy(), self.s.s8.reshape(-1)[: fl.blocks(cols) * ROWS].reshape(-1, ROWS).cpu().numpy()

    def plan(self):
        s = self.s
        assert s.status.tolist()[0] == 0
        self.old = (s.lens.cpu().numpy() - s.new.cpu().numpy()).tolist()
        masks, positions = tl.plan(self.shapes, WORDS, ROWS, s.lens.tolist(), np.zeros((ROWS, WORDS), np.uint32), np.zeros(ROWS, np.uint32))
        n = self.used()
        trees = np.repeat([not isinstance(x, int) for x in self.shapes], s.new.tolist())
        assert np.array_equal(s.masks[:n].cpu().numpy().view(np.uint32)[trees], masks[:n][trees])
        assert np.array_equal(s.positions[:n].cpu().numpy().view(np.uint32), positions[:n])

    def quantize(self, x, cols):
        q, scales = fl.quantize(x[:, :cols].float().cpu().numpy())
        got = self.codes(cols)
        assert np.array_equal(got[0], q) and np.array_equal(got[1], scales)

    def products(self, w, dtype):
        return fl.product(*self.codes(w[0].shape[1]), w[0], w[1].astype(np.float32), dtype)

    def gemm(self, w, y, dtype, res):
        want, tol = self.products(w, dtype)
        if res is not None:
            want = want + res.double().cpu().numpy()
            tol = tol + np.abs(want) * 2.0 ** -24
        fl.near(y.double().cpu().numpy(), want, tol, dtype)

    def gateup(self, l, y):
        want, tol = fl.gated(*self.products(l["gate"], arc.BF16), *self.products(l["up"], arc.BF16), arc.BF16)
        fl.near(y.double().cpu().numpy(), want, tol, arc.BF16)

    def attention(self, l):
        s = self.s
        tables, starts, lens = s.tables.cpu().numpy(), s.starts.tolist(), s.lens.tolist()
        q, out = (t.double().cpu().numpy().reshape(ROWS, HEADS, DIM) for t in (s.q, s.attn))
        for b, shape in enumerate(self.shapes):
            pos = np.arange(lens[b])
            K, V = (t.cpu().numpy()[tables[b, pos // PAGE], pos % PAGE].astype(np.float64) for t in l["kv"])
            for i in range(starts[b + 1] - starts[b]):
                see = pos < self.old[b]
                see[[self.old[b] + j for j in (range(i + 1) if isinstance(shape, int) else tl.ancestors(shape, i))]] = True
                ref, mass, off, seen = tl.attend_seen(q[starts[b] + i], K, V, see, DIM ** -0.5)
                tol = pl.attention_bound(ref, mass, off, seen, np.abs(V).max(), arc.F16)
                assert np.all(np.abs(out[starts[b] + i] - ref) <= tol), (b, i)

    def before_commit(self):
        s = self.s
        said = np.array([tl.argmax(r) for r in s.logits.cpu().numpy()], np.uint32)
        pools = [tuple(t.cpu().numpy().view(np.uint16) for t in l["kv"]) for l in s.layers]
        self.want = tl.commit(self.shapes, WORDS, s.lens.cpu().numpy().view(np.uint32), s.starts.cpu().numpy(), s.tables.cpu().numpy(), PAGE,
                              s.drafts.cpu().numpy().view(np.uint32), said, pools, s.stack.cpu().numpy().view(np.uint32), int(s.count), POOL)

    def after(self):
        torch.cuda.synchronize()
        s, w, n = self.s, self.want, self.used()
        assert s.counts.tolist() == w["counts"].tolist() and s.lens.tolist() == w["lens"].tolist()
        assert np.array_equal(s.tokens[:n].cpu().numpy().view(np.uint32), w["tokens"][:n])
        assert int(s.count) == w["count"] and np.array_equal(s.stack.cpu().numpy().view(np.uint32)[: w["count"]], w["stack"][: w["count"]])
        for l, (k, v) in zip(s.layers, w["pools"]):
            assert all(np.array_equal(t.cpu().numpy().view(np.uint16), want) for t, want in zip(l["kv"], (k, v)))
        # every page is free or holds positions of one request
        held = [pl.pages_of(x, PAGE) for x in s.lens.tolist()]
        ids = [int(i) for b, h in enumerate(held) for i in s.tables[b, :h]] + s.stack[: int(s.count)].tolist()
        assert sorted(ids) == list(range(POOL))


def some_trees(rng, last):
    """Trees whose node 0 is each request's last token, many children, so that some are accepted."""
    shapes = [[tl.NONE] + [int(rng.integers(0, max(1, i // 2))) for i in range(1, int(n))] for n in rng.integers(1, 21, B)]
    tokens = rng.integers(0, VOCAB, sum(map(len, shapes)))
    at = 0
    for b, s in enumerate(shapes):
        tokens[at] = last[b]
        at += len(s)
    return shapes, tokens


def test_steps_of_a_server():
    rng = np.random.default_rng(SEED + 1)
    s = Server()
    check = Check(s)
    # prompts: one longer than a tree's words hold, which is a chunk, two short ones as chains
    check.shapes = [40, tl.chain(9), tl.chain(1)]
    tokens = rng.integers(0, VOCAB, 50)
    s.draft(check.shapes, tokens)
    s.step(check)
    check.after()
    accepted = 0
    for _ in range(4):
        starts = s.starts.tolist()
        last = [int(s.tokens[starts[b] + int(s.counts[b]) - 1]) for b in range(B)]
        check.shapes, tokens = some_trees(rng, last)
        s.draft(check.shapes, tokens)
        s.step(check)
        check.after()
        accepted += int(s.counts.sum()) - B
    assert accepted > 0 and check.seen == {"plan", "quantize", "gemm", "attention", "gateup", "before commit"}


def test_captured_step_replays():
    """The whole step captured once and replayed with other trees: each replay equals the eager step of a second
    server, with eager work and synchronizations between the replays."""
    rng = np.random.default_rng(SEED + 2)
    a, b = Server(), Server()
    shapes, tokens = some_trees(rng, [1, 2, 3])
    for s in (a, b):
        s.draft(shapes, tokens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    torch.cuda.synchronize()
    for i in range(5):
        shapes, tokens = some_trees(rng, rng.integers(0, VOCAB, B))
        for s in (a, b):
            s.draft(shapes, tokens)
        b.step()
        g.replay()
        torch.cuda.synchronize()
        assert a.status.tolist()[0] == 0
        for name in Server.STATE:
            assert torch.equal(getattr(a, name), getattr(b, name)), (i, name)
        for x, y in zip(a.layers, b.layers):
            assert torch.equal(x["kv"][0], y["kv"][0]) and torch.equal(x["kv"][1], y["kv"][1])
    assert int(a.lens.min()) >= 5


def test_two_captured_steps_side_by_side():
    """Two graphs, each with its own buffers and workspace, replayed at once on two streams."""
    servers, graphs, streams = [], [], []
    rng = np.random.default_rng(SEED + 3)
    shapes, tokens = some_trees(rng, [4, 5, 6])
    for _ in range(2):
        s = Server()
        s.draft(shapes, tokens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.step()
        servers.append(s)
        graphs.append(g)
        streams.append(torch.cuda.Stream())
    c = Server()
    c.draft(shapes, tokens)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    for _ in range(3):
        c.step()
    torch.cuda.synchronize()
    for s in servers:
        for name in Server.STATE:
            assert torch.equal(getattr(s, name), getattr(c, name)), name


@pytest.mark.parametrize("logits", [False, True])
def test_captured_commit_of_one_request(logits):
    """One request's step end with lens_out apart from lens, captured once and replayed with other drafts, trees and
    lengths: each replay equals the eager call on a second set of buffers."""
    rng = np.random.default_rng(SEED + 4)
    n, layers, vocab = 40, 5, 50

    class Side:
        def __init__(self):
            self.kv = [[torch.arange(20 * PAGE * KV * DIM, device="cuda").remainder(2000 + 7 * i + j).half().view(20, PAGE, KV, DIM) for j in range(2)]
                       for i in range(layers)]
            self.tables = torch.randperm(20, generator=torch.Generator().manual_seed(1)).int().cuda().view(1, 20)
            self.lens, self.starts = i32(1), i32(2)
            self.parents, self.drafts, self.targets, self.tokens = i32(n), i32(n), i32(n), i32(n)
            self.lens_out, self.counts, self.stack, self.count, self.count_out = i32(1), i32(1), i32(20), i32(1, fill=2), i32(1)
            self.logits = torch.zeros(n, vocab, device="cuda")
            self.pages = [arc.KvPages(p(k), p(v), 20, PAGE, KV, DIM, arc.F16) for k, v in self.kv]
            self.batch = arc.PagedBatch(1, n, 20, n, p(self.tables), p(self.lens), p(self.starts))
            self.ws = torch.full((arc.tree_commit_workspace_bytes(self.batch),), 255, dtype=torch.uint8, device="cuda")

        def commit(self):
            more = dict(logits=p(self.logits), ldl=vocab, vocab=vocab) if logits else {}
            arc.tree_commit(self.pages, self.batch, arc.Tree(p(self.parents), None, 2), p(self.drafts), p(self.targets), p(self.lens_out),
                            p(self.counts), p(self.tokens), p(self.ws), free_pages=p(self.stack), num_pages=20, free_count=p(self.count),
                            free_count_out=p(self.count_out), stream=TorchStream(), **more)

    a, b = Side(), Side()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.commit()
    torch.cuda.synchronize()
    moved = 0
    for rows in (40, 33, 1, 40):
        parents = tl.random_tree(rng, rows) + [tl.NONE] * (n - rows)
        said = rng.integers(0, vocab, n)
        drafts = [int(said[q]) if q < i and rng.random() < 0.9 else 3 for i, q in enumerate(parents)]
        x = rng.standard_normal((n, vocab)).astype(np.float32)
        x[np.arange(n), said] = 9.0
        length = int(rng.integers(0, 20 * PAGE - n)) + rows
        for s in (a, b):
            for dst, src in ((s.parents, np.array(parents, np.uint32).view(np.int32)), (s.drafts, np.array(drafts, np.int32)),
                             (s.targets, said.astype(np.int32)), (s.lens, np.array([length], np.int32)), (s.starts, np.array([0, rows], np.int32)),
                             (s.logits, x)):
                dst.copy_(torch.from_numpy(src))
        b.commit()
        g.replay()
        torch.cuda.synchronize()
        for name in ("lens_out", "counts", "tokens", "targets", "stack", "count_out"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
        assert all(torch.equal(x, y) for u, v in zip(a.kv, b.kv) for x, y in zip(u, v))
        assert 1 <= int(a.counts) <= rows and int(a.lens_out) == length - rows + int(a.counts)
        moved += int(a.counts) - 1
    assert moved > 0


@pytest.mark.parametrize("dim", [64, 128])
def test_a_chain_is_a_chunk(dim):
    """A tree that is a chain sees what a causal chunk sees: tree attention of both, and paged attention, on the same rows."""
    old, n = [500, 33], [30, 32]
    chain = tl.TreeStep(old, [tl.chain(x) for x in n], 16, 2, 7, dim, arc.F16, SEED).upload()
    chain.check(chain.attention())
    pl.Step.check(chain, pl.Step.attention(chain))


def test_what_is_accepted_is_what_a_chunk_of_it_would_be():
    """The accepted nodes' outputs, and those of their tokens as a causal chunk over the committed cache, are the same rows of
    float64."""
    rng = np.random.default_rng(SEED + 5)
    old, tree = 70, tl.random_tree(rng, 30)
    s = tl.TreeStep([old], [tree], 16, 2, 4, 128, arc.F16, SEED + 6).upload()
    bits = s.attention()
    path = [0]
    while True:
        child = [i for i in range(len(tree)) if tree[i] == path[-1]]
        if not child:
            break
        path.append(child[-1])
    drafts, targets = np.zeros(30, np.uint32), np.full(30, 99, np.uint32)
    for a, b in zip(path, path[1:]):
        drafts[b] = targets[a] = b
    D = arc.DeviceBuffer.from_array
    out = [arc.DeviceBuffer(4 * 40) for _ in range(2)]
    ws = arc.DeviceBuffer(arc.tree_commit_workspace_bytes(s.batch))
    arc.tree_commit([s.pages], s.batch, s.tree, D(drafts), D(targets), s.dlens, out[0], out[1], ws)
    k = len(path)
    assert k > 3 and s.dlens.download(np.uint32).tolist() == [old + k] and out[0].download(np.uint32, 1).tolist() == [k]
    q = D(s.q[path])
    starts = D(np.array([0, k], np.uint32))
    chunk = arc.PagedBatch(1, k, s.max_pages, k, s.dtables, s.dlens, starts)
    got = D(np.zeros((k, s.ldo), np.uint16))
    space = arc.DeviceBuffer(arc.paged_attention_workspace_bytes(s.pages, chunk, s.hpk))
    arc.paged_attention(s.pages, chunk, q, s.ldq, s.hpk, got, s.ldo, space)
    s.check(bits)
    rows = pl.from_bits(got.download(np.uint16).reshape(k, s.ldo)[:, : s.width], arc.F16).reshape(k, s.heads, s.dim)
    for i, node in enumerate(path):  # the same keys and values, now side by side
        q = pl.from_bits(s.q[node, : s.width], arc.F16).reshape(s.heads, s.dim)
        ref, mass, off, seen = tl.attend_seen(q, s.K[0], s.V[0], s.seen(0, node), s.dim ** -0.5)
        assert np.all(np.abs(rows[i] - ref) <= pl.attention_bound(ref, mass, off, seen, np.abs(s.V[0]).max(), arc.F16)), i
