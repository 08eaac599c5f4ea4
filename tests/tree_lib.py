"""Float64 and whole-number statements of the draft-tree entry points, and random steps with trees to hold
them to: masks and positions from parents, what each row sees, the walk, the rows' move."""
import numpy as np

import arcllm_amd as arc
import paged_lib as pl

U32 = np.uint32
NONE = arc.NO_PARENT


# -------------------------------------------------------------------- trees
def chain(n):
    return [NONE] + list(range(n - 1))


def star(n):
    return [NONE] + [0] * (n - 1)


def random_tree(rng, n, roots=0.0):
    return [NONE] + [NONE if rng.random() < roots else int(rng.integers(max(0, (i - 1) // 3), i)) for i in range(1, n)]


def ancestors(parents, i):
    """Node i and those it descends from, deepest first; a parent that is not before its node is none."""
    out = [i]
    while parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def mask_words(nodes, words):
    m = np.zeros(words, U32)
    for j in nodes:
        m[j >> 5] |= U32(1 << (j & 31))
    return m


def plan(shapes, words, rows, lens, masks, positions):
    """What arc_tree_plan leaves: shapes[b] is a list of parents, or a number of rows (a chunk)."""
    masks, positions, at = masks.copy(), positions.copy(), 0
    for shape, held in zip(shapes, lens):
        n = shape if isinstance(shape, int) else len(shape)
        base = max(0, held - n)
        for i in range(min(n, rows - at)):
            if min(n, rows - at) > 32 * words:
                positions[at + i] = base + i
                continue
            up = ancestors(shape if not isinstance(shape, int) else chain(n), i)
            masks[at + i] = mask_words(up, words)
            positions[at + i] = base + len(up) - 1
        at = min(rows, at + n)
    return masks, positions


# ---------------------------------------------------------------- attention
def attend_seen(q, K, V, see, scale):
    """paged_lib.attend for a row that sees the positions `see`."""
    heads, D = q.shape
    hpk = heads // K.shape[1]
    if not see.any():
        return np.zeros_like(q), np.zeros_like(q), 0.0, 0
    k, v = K[see].repeat(hpk, 1), V[see].repeat(hpk, 1)
    s = np.einsum("hd,jhd->hj", q, k) * scale
    off = np.einsum("hd,jhd->hj", np.abs(q), np.abs(k)).max() * scale * (D + 2) * 2.0 ** -24
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return np.einsum("hj,jhd->hd", p, v), np.einsum("hj,jhd->hd", p, np.abs(v)), off, int(see.sum())


class TreeStep(pl.Step):
    """A step whose requests hold trees (lists of parents) or chunks (numbers of rows); masks[row], if given for
    a row, replaces the tree's."""

    def __init__(self, old, shapes, *args, words=None, masks=None, **kw):
        new = [s if isinstance(s, int) else len(s) for s in shapes]
        super().__init__(old, new, *args, **kw)
        self.shapes = shapes
        trees = [len(s) for s in shapes if not isinstance(s, int)]
        self.words = words or max(1, -(-max(trees, default=1) // 32))
        assert all(n <= 32 * self.words for n in trees) and all(s > 32 * self.words for s in shapes if isinstance(s, int))
        self.parents = np.full(max(1, self.rows), NONE, U32)
        at = 0
        for s, n in zip(shapes, new):
            if not isinstance(s, int):
                self.parents[at: at + n] = s
            at += n
        self.custom = masks or {}

    def upload(self):
        super().upload()
        D = arc.DeviceBuffer.from_array
        rows = max(1, self.rows)
        self.dparents, self.dpositions = D(self.parents), D(np.full(rows, 0xFFFFFFFF, U32))
        self.dmasks = D(np.full((rows, self.words), 0xFFFFFFFF, U32))
        self.batch = arc.PagedBatch(len(self.old), self.rows, self.max_pages, self.max_new, self.dtables, self.dlens,
                                    self.dstarts, self.dpositions)
        self.tree = arc.Tree(self.dparents, self.dmasks, self.words)
        arc.tree_plan(self.batch, self.tree)
        if self.custom:
            m = self.dmasks.download(U32).reshape(rows, self.words)
            for row, nodes in self.custom.items():
                m[row] = mask_words(nodes, self.words)
            self.dmasks.upload(m)
        return self

    def attention(self, scale=0.0, window=0, sinks=0, workspace=None, stream=None):
        out = arc.DeviceBuffer.from_array(np.full((max(1, self.rows), self.ldo), 0xABCD, np.uint16))
        ws = workspace or arc.DeviceBuffer(arc.tree_attention_workspace_bytes(self.pages, self.batch, self.hpk))
        if workspace is None:
            ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
        arc.tree_attention(self.pages, self.batch, self.tree, self.dq, self.ldq, self.hpk, out, self.ldo, ws, scale=scale,
                           window=window, sinks=sinks, stream=stream)
        if stream is not None:
            stream.synchronize()
        return out.download(np.uint16).reshape(-1, self.ldo)[: self.rows]

    def seen(self, b, i, window=0, sinks=0):
        """The positions that row i of request b sees."""
        old, shape, n = self.old[b], self.shapes[b], self.new[b]
        see = np.arange(old + n) < old
        place = np.arange(old + n)
        if isinstance(shape, int):
            see[old: old + i + 1] = True
            pos = old + i
        else:
            row = int(self.starts[b]) + i
            nodes = sorted(j for j in self.custom.get(row, ancestors(shape, i)) if j <= i)
            see[[old + j for j in nodes]] = True
            place[[old + j for j in nodes]] = old + np.arange(len(nodes))
            pos = old + len(ancestors(shape, i)) - 1
        return see & ((pos - place < window) | (place < sinks)) if window else see

    def check(self, bits, scale=0.0, window=0, sinks=0, rows=None, dropped=None):
        s = scale or self.dim ** -0.5
        worst = 0.0
        assert np.all(bits[self.used:] == 0xABCD), "rows behind the last request"
        assert np.all(bits[:, self.width:] == 0xABCD), "columns behind the heads"
        for b, n in enumerate(self.new):
            vmax = np.abs(self.V[b][np.isfinite(self.V[b])]).max() if len(self.V[b]) else 0.0
            for i in range(n):
                row = int(self.starts[b]) + i
                if rows is not None and row not in rows:
                    continue
                q = pl.from_bits(self.q[row, : self.width], self.dtype).reshape(self.heads, self.dim)
                see = self.seen(b, i, window, sinks)
                if dropped is not None:
                    see &= ~dropped[b]
                ref, mass, off, seen = attend_seen(q, self.K[b], self.V[b], see, s)
                got = pl.from_bits(bits[row, : self.width], self.dtype).reshape(self.heads, self.dim)
                tol = pl.attention_bound(ref, mass, off, seen, vmax, self.dtype)
                assert np.all(np.isfinite(got)), (b, i)
                share = float((np.abs(got - ref) / tol).max())
                assert share <= 1.0, (b, i, share, float(np.abs(got - ref).max()))
                worst = max(worst, share)
        return worst


# ------------------------------------------------------------------- commit
def argmax(row):
    """The largest, the lowest of equals; NaN never; 0 without a number."""
    best, at = -np.inf, None
    for i, v in enumerate(row):
        if v > best or (v == best and at is None):
            best, at = v, i
    return 0 if at is None else at


def walk(parents, drafts, targets):
    """Nodes from 0 on, each the first child that holds the target's token after its parent."""
    path = [0]
    while True:
        node = path[-1]
        child = [i for i in range(node + 1, len(parents)) if parents[i] == node and drafts[i] == targets[node]]
        if not child:
            return path
        path.append(child[0])


def commit(shapes, words, lens, starts, tables, page, drafts, targets, pools, stack, count, num_pages):
    """What arc_tree_commit leaves.  pools: per layer (k, v), each [pages][positions][values]."""
    pools = [(k.copy(), v.copy()) for k, v in pools]
    stack, lens_out, counts = stack.copy(), lens.copy(), np.zeros(len(shapes), U32)
    tokens = np.full(len(drafts), arc.NO_TOKEN, U32)
    pages = len(pools[0][0])
    for b, shape in enumerate(shapes):
        n, at = shape if isinstance(shape, int) else len(shape), int(starts[b])
        if n == 0:
            continue
        if n > 32 * words:
            counts[b], tokens[at] = 1, targets[at + n - 1]
            continue
        path = walk(shape, drafts[at: at + n], targets[at: at + n])
        counts[b], base = len(path), int(lens[b]) - n
        tokens[at: at + len(path)] = [targets[at + i] for i in path]
        lens_out[b] = base + len(path)
        for to, of in enumerate(path):
            ends = [tables[b][(base + x) // page] for x in (to, of)]
            if max(ends) < pages:
                for k, v in pools:
                    for t in (k, v):
                        t[ends[0], (base + to) % page] = t[ends[1], (base + of) % page]
        for p in range(pl.pages_of(int(lens_out[b]), page), pl.pages_of(int(lens[b]), page)):
            if count < num_pages:
                stack[count] = tables[b][p]
                count += 1
    return dict(counts=counts, tokens=tokens, lens=lens_out, pools=pools, stack=stack, count=count)
