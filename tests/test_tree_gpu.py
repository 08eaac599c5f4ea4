"""The draft-tree entry points on the GPU: masks, positions and commits bit for bit, attention against float64."""
import numpy as np
import pytest
import torch

import arcllm_amd as arc
import paged_lib as pl
import tree_lib as tl

pytestmark = pytest.mark.gpu

SEED = 0x7AEE
D = arc.DeviceBuffer.from_array
U32 = np.uint32
TYPES = [arc.F16, arc.BF16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


def rng_of(*key):
    return np.random.default_rng([SEED, *key])


# --------------------------------------------------------------------- plan
def run_plan(shapes, words, old, rows=None, lens=None):
    new = [s if isinstance(s, int) else len(s) for s in shapes]
    starts = np.concatenate([[0], np.cumsum(new)]).astype(U32)
    rows = int(starts[-1]) if rows is None else rows
    lens = [o + n for o, n in zip(old, new)] if lens is None else lens
    parents = np.concatenate([np.zeros(0, U32)] + [np.full(s, 7, U32) if isinstance(s, int) else np.array(s, U32) for s in shapes])
    parents = np.concatenate([parents, np.full(max(1, rows), 3, U32)])[: max(1, rows)]
    masks, positions = np.full((max(1, rows), words), 0xABABABAB, U32), np.full(max(1, rows), 0xCDCDCDCD, U32)
    d = [D(x) for x in (np.array(lens + [0], U32), starts, parents, masks, positions)]
    batch = arc.PagedBatch(len(shapes), rows, lens=d[0], starts=d[1], positions=d[4])
    arc.tree_plan(batch, arc.Tree(d[2], d[3], words))
    want = tl.plan(shapes, words, rows, lens, masks, positions)
    got = d[3].download(U32).reshape(masks.shape), d[4].download(U32)
    assert np.array_equal(got[1][:rows], want[1][:rows]) and np.array_equal(got[0][:rows], want[0][:rows])


@pytest.mark.parametrize("words", [1, 2, 3, 8, 32])
@pytest.mark.parametrize("kind", ["chain", "star", "random", "roots"])
def test_plan_trees(kind, words):
    rng = rng_of(words)
    sizes = sorted({1, 2, 31, 32, 32 * words - 1, 32 * words, max(1, 17 * words)} - {n for n in (31, 32) if n > 32 * words})
    make = dict(chain=tl.chain, star=tl.star, random=lambda n: tl.random_tree(rng, n), roots=lambda n: tl.random_tree(rng, n, 0.3))[kind]
    run_plan([make(n) for n in sizes], words, [int(x) for x in rng.integers(0, 5000, len(sizes))], rows=sum(sizes) + 5)


def test_plan_parents_that_are_none():
    # itself, one behind it, numbers far out of range
    run_plan([[5, 1, 9, 0, 0xFFFFFFF0, 3, 6], [0], [1, 0]], 1, [10, 0, 3])


def test_plan_mixed_chunks_and_empty_requests():
    rng = rng_of(3)
    shapes = [tl.random_tree(rng, 20), 33, [], tl.chain(1), 700, tl.random_tree(rng, 32), []]
    run_plan(shapes, 1, [0, 5, 9, 77, 0, 2 ** 31 - 100, 4], rows=800)


def test_plan_rows_that_the_step_does_not_have():
    rng = rng_of(4)
    run_plan([tl.random_tree(rng, 20), tl.chain(30), tl.chain(5)], 1, [3, 4, 5], rows=32)  # a tree cut, one left out
    run_plan([tl.chain(8)], 1, [0], lens=[5])  # fewer positions than rows
    run_plan([40], 1, [0], rows=36, lens=[40])


def test_plan_many_requests():
    rng = rng_of(5)
    shapes = [tl.random_tree(rng, int(n)) for n in rng.integers(0, 33, 3000) if n]
    run_plan(shapes, 2, rng.integers(0, 10 ** 6, len(shapes)).tolist())


def test_plan_twice_over_itself():
    rng = rng_of(6)
    s = tl.TreeStep([40, 3], [tl.random_tree(rng, 25), tl.chain(4)], 16, 1, 1, 64, arc.F16, 1).upload()
    first = s.dmasks.download(U32), s.dpositions.download(U32)
    arc.tree_plan(s.batch, s.tree)
    assert np.array_equal(first[0], s.dmasks.download(U32)) and np.array_equal(first[1], s.dpositions.download(U32))


# ---------------------------------------------------------------- attention
def check(old, shapes, page=16, kv_heads=2, hpk=4, dim=128, dtype=arc.F16, seed=0, window=0, sinks=0, **kw):
    s = tl.TreeStep(old, shapes, page, kv_heads, hpk, dim, dtype, SEED + seed, **kw).upload()
    s.check(s.attention(window=window, sinks=sinks), window=window, sinks=sinks)
    return s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,hpk", [(1, 1), (4, 7), (2, 8), (3, 5), (1, 33), (1, 64)])
def test_heads(kv_heads, hpk, dim, dtype):
    rng = rng_of(kv_heads, hpk)
    check([37, 0, 130], [tl.random_tree(rng, 19), tl.random_tree(rng, 5), tl.chain(1)], kv_heads=kv_heads, hpk=hpk, dim=dim, dtype=dtype)


@pytest.mark.parametrize("n", [1, 2, 4, 5, 8, 9, 16, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 250])
@pytest.mark.parametrize("old", [0, 1, 31, 32, 77])
def test_tree_sizes(n, old):
    check([old], [tl.random_tree(rng_of(n, old), n)], kv_heads=1, seed=n, words=-(-n // 32))


@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
@pytest.mark.parametrize("dim", [64, 128])
def test_tree_kinds(kind, dim):
    make = dict(chain=tl.chain, star=tl.star, roots=lambda n: tl.random_tree(rng_of(2), n, 0.4))[kind]
    check([90, 500, 3], [make(40), make(64), make(7)], dim=dim, hpk=6)


def test_the_largest_tree():
    check([100], [tl.random_tree(rng_of(1), 1024)], kv_heads=1, hpk=1, dim=64, words=32)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 1024, 65536])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_sizes(page, dim):
    rng = rng_of(page)
    check([0, 60, 300], [tl.random_tree(rng, 33), tl.random_tree(rng, 3), tl.random_tree(rng, 20)], page=page, dim=dim, spare=1)


@pytest.mark.parametrize("old", [16, 100, 511, 512, 513, 1000, 2047, 5000])
@pytest.mark.parametrize("n", [3, 26])
def test_context_lengths(old, n):
    check([old], [tl.random_tree(rng_of(old), n)], kv_heads=2, hpk=7, dtype=arc.BF16)


def test_ragged_batch_rows_behind_and_strides():
    rng = rng_of(8)
    old = rng.integers(0, 400, 21).tolist()
    shapes = [tl.random_tree(rng, int(n)) for n in rng.integers(1, 60, 21)]
    shapes[3], shapes[7], old[7] = [], tl.chain(1), 0
    check(old, shapes, hpk=3, rows=sum(map(len, shapes)) + 11, stride_pad=64, ld_pad=24, max_pages=40)


@pytest.mark.parametrize("hpk", [1, 4])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_beside_trees(dim, hpk):
    rng = rng_of(9)
    s = check([70, 0, 300, 12], [tl.random_tree(rng, 20), 45, tl.chain(1), 130], dim=dim, hpk=hpk, words=1)
    # a step of chunks alone is paged attention, bit for bit where it takes the same kernels
    s = tl.TreeStep([70, 0], [200, 340], 16, 2, 4, dim, arc.F16, 3, words=1).upload()
    bits = s.attention()
    s.check(bits)
    assert np.array_equal(bits, pl.Step.attention(s))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (5, 2), (7, 90), (33, 0), (64, 4), (100, 65), (128, 700), (1000, 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_window_and_sinks(window, sinks, dim):
    rng = rng_of(window, sinks)
    # windows shorter than a tree is deep, sinks that reach into the tree, chunks beside
    shapes = [tl.chain(40), tl.random_tree(rng, 50), tl.random_tree(rng, 3), 70, tl.chain(1)]
    check([80, 300, 2, 150, 400], shapes, dim=dim, window=window, sinks=sinks, words=2)


def test_window_far_behind():
    rng = rng_of(10)
    check([9000, 5000], [tl.random_tree(rng, 30), tl.chain(20)], kv_heads=1, hpk=7, window=512, sinks=4)


def test_masks_of_the_callers_own():
    # rows that see nothing of the step, all before them, bits above their own place, which do not count
    n = 40
    masks = {0: [], 3: [], 7: list(range(n)), 20: list(range(0, n, 3)), 39: list(range(n)), 38: [39]}
    s = check([50], [tl.star(n)], masks=masks, hpk=5)
    # nothing at all to see: zeros
    s = tl.TreeStep([0], [tl.star(9)], 16, 1, 4, 64, arc.F16, 2, masks={0: [], 4: []}).upload()
    bits = s.attention()
    s.check(bits)
    assert not bits[0, : s.width].any() and not bits[4, : s.width].any() and bits[1, : s.width].any()


def test_scale_sign_and_size():
    for scale in (0.02, 1.0):
        s = tl.TreeStep([200, 3], [tl.random_tree(rng_of(11), 30), tl.chain(2)], 16, 2, 4, 128, arc.F16, 4).upload()
        s.check(s.attention(scale=scale), scale=scale)


def poison(s, b, positions, value):
    """Sets K and V at positions of request b."""
    for p in positions:
        place = (p % s.page) * s.kvd
        at = s.tables[b, p // s.page], slice(place, place + s.kvd)
        s.k[at] = s.v[at] = value


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [0x7C00, 0xFC00, 0x7E00])
def test_infinities_and_nan_in_nodes_that_a_row_does_not_see(bits, dim):
    # nodes 3 and 17 hold them; rows that see neither are as without
    shapes = [tl.star(24), tl.random_tree(rng_of(12), 30)]
    s = tl.TreeStep([70, 10], shapes, 16, 2, 4, dim, arc.F16, 6)
    hidden = {0: [3, 17], 1: [29]}
    for b, nodes in hidden.items():
        poison(s, b, [s.old[b] + j for j in nodes], bits)
    s.upload()
    got = s.attention()
    sees = {int(s.starts[b]) + i for b, nodes in hidden.items() for i in range(s.new[b]) if set(nodes) & set(tl.ancestors(shapes[b], i))}
    keep = [r for r in range(s.rows) if r not in sees]
    s.check(got, rows=set(keep))
    for row in sees:  # the row's own node is one of them: its key's score is infinite or NaN
        assert not np.all(np.isfinite(pl.from_bits(got[row, : s.width], arc.F16)))


def test_pages_outside_the_pool_are_not_read():
    s = tl.TreeStep([100, 40], [tl.random_tree(rng_of(13), 40), tl.chain(9)], 8, 2, 4, 128, arc.F16, 7)
    dropped = [np.zeros(140, bool), np.zeros(49, bool)]
    for b, entry in ((0, 2), (0, 15), (1, 5)):
        s.tables[b, entry] = s.num_pages + entry
        dropped[b][entry * 8: entry * 8 + 8] = True
    s.upload()
    s.check(s.attention(), dropped=dropped)


def test_starts_beyond_the_rows_and_short_lens():
    s = tl.TreeStep([30, 20], [tl.chain(10), tl.chain(20)], 16, 1, 4, 64, arc.F16, 8)
    s.upload()
    full = s.attention()
    s.batch.tokens = 18  # the second tree's last 12 rows are not there
    s.rows = 18
    arc.tree_plan(s.batch, s.tree)
    cut = s.attention()
    assert np.array_equal(cut, full[:18])
    # fewer positions than rows: nodes without a place are not there
    s = tl.TreeStep([0], [tl.chain(12)], 16, 1, 4, 64, arc.F16, 8)
    s.lens[:] = 5
    s.upload()
    assert np.all(np.isfinite(pl.from_bits(s.attention(), arc.F16)))


def test_long_context_offsets_pass_32_bits():
    """Pages 2^31 elements and more from the pool's start."""
    dim, kv_heads, page, far = 64, 1, 16, 1 << 22
    stride = 1 << 11
    n_pages = far + 2
    k = torch.zeros(n_pages * stride, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    rng = rng_of(14)
    old, parents = 20, tl.random_tree(rng, 9)
    ids = np.array([[far + 1, far]], U32)
    K, V = (pl.to_bits(rng.standard_normal((29, dim)), arc.F16) for _ in range(2))
    for pool, rows in ((k, K), (v, V)):
        for p in range(29):
            at = int(ids[0, p // page]) * stride + (p % page) * dim
            pool[at: at + dim] = torch.from_numpy(rows[p].view(np.float16)).cuda()
    s = tl.TreeStep([old], [parents], page, kv_heads, 4, dim, arc.F16, 3)
    s.upload()
    s.dtables.upload(np.pad(ids, ((0, 0), (0, s.max_pages - 2))))
    s.pages = arc.KvPages(k.data_ptr(), v.data_ptr(), n_pages, page, kv_heads, dim, arc.F16, stride)
    s.K, s.V = ([pl.from_bits(x, arc.F16).reshape(29, 1, dim)] for x in (K, V))
    torch.cuda.synchronize()
    s.check(s.attention())


@pytest.mark.parametrize("dtype", TYPES)
def test_many_trees(dtype):
    rng = rng_of(15)
    old = rng.integers(0, 300, 300).tolist()
    check(old, [tl.random_tree(rng, int(n)) for n in rng.integers(1, 12, 300)], kv_heads=1, hpk=7, dtype=dtype)


@pytest.mark.parametrize("kv_heads,hpk", [(1, 4), (4, 7)])
@pytest.mark.parametrize("most", [0, 3, 130])
def test_many_short_contexts(most, kv_heads, hpk):
    rng = rng_of(11, most)
    check(rng.integers(0, most + 1, 41).tolist(), [tl.random_tree(rng, int(n)) for n in rng.integers(1, 5, 41)], kv_heads=kv_heads, hpk=hpk)


def test_many_requests_of_one_row_and_few_trees():
    rng = rng_of(16)
    shapes = [tl.chain(1)] * 150
    shapes[20], shapes[149] = tl.random_tree(rng, 60), tl.random_tree(rng, 33)
    check(rng.integers(0, 200, 150).tolist(), shapes, kv_heads=2, hpk=4)


def test_same_call_twice_gives_the_same_bits():
    rng = rng_of(17)
    s = tl.TreeStep([3000, 200, 7000], [tl.random_tree(rng, 40) for _ in range(3)], 16, 4, 7, 128, arc.F16, 9).upload()
    assert np.array_equal(s.attention(), s.attention())


def test_long_context_is_split():
    s = tl.TreeStep([40000], [tl.random_tree(rng_of(18), 26)], 64, 2, 7, 128, arc.BF16, 10).upload()
    s.check(s.attention(), rows={0, 1, 13, 25})


# ------------------------------------------------------------------- commit
class CommitRun:
    def __init__(self, old, shapes, page=16, kv_heads=2, dim=64, dtype=arc.F16, layers=2, words=None, spare=3, seed=0, rows=0,
                 vocab=50, agree=0.7, stride_pad=0, count=2):
        rng = rng_of(seed)
        self.shapes, self.page = shapes, page
        new = [s if isinstance(s, int) else len(s) for s in shapes]
        self.words = words or max(1, -(-max([len(s) for s in shapes if not isinstance(s, int)], default=1) // 32))
        self.lens = np.array([o + n for o, n in zip(old, new)], U32)
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(U32)
        self.used, self.rows = sum(new), sum(new) + rows
        need = [pl.pages_of(int(n), page) for n in self.lens]
        self.pool = sum(need) + spare
        order = rng.permutation(self.pool).astype(U32)
        self.max_pages = max(1, max(need, default=1))
        self.tables = np.full((max(1, len(old)), self.max_pages), 0xFFFFFFFF, U32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at: at + n]
            at += n
        self.kvd, self.stride_pad, self.layers = kv_heads * dim, stride_pad, layers
        self.kv = rng.integers(0, 2 ** 16, (layers, 2, self.pool, page * self.kvd + stride_pad), dtype=np.uint16)
        self.stack = np.full(self.pool, 0xEEEEEEEE, U32)
        self.stack[:count] = order[at: at + count]
        self.count = count
        self.parents = np.concatenate([np.zeros(0, U32)] + [np.full(s, 9, U32) if isinstance(s, int) else np.array(s, U32) for s in shapes]
                                      + [np.zeros(rows + 1, U32)])
        self.targets = rng.integers(0, vocab, self.rows + 1).astype(U32)
        self.drafts = rng.integers(0, vocab, self.rows + 1).astype(U32)
        for b, s in enumerate(shapes):  # most drafts are what the target says after their parent
            for i in range(1, new[b] if not isinstance(s, int) else 0):
                if s[i] < i and rng.random() < agree:
                    self.drafts[self.starts[b] + i] = self.targets[self.starts[b] + s[i]]
        self.vocab, self.dims = vocab, (kv_heads, dim, dtype)

    def run(self, logits=None, ldl=0, dtype=arc.F32, in_place=False, free_list=True, num_pages=None, stream=None):
        B = len(self.shapes)
        self.dkv = D(self.kv)
        size = self.kv[0, 0].nbytes
        kv_heads, dim, dt = self.dims
        layers = [arc.KvPages(self.dkv.ptr + 2 * i * size, self.dkv.ptr + (2 * i + 1) * size, self.pool, self.page, kv_heads, dim, dt,
                              self.page * self.kvd + self.stride_pad) for i in range(self.layers)]
        d = {k: D(v) for k, v in dict(tables=self.tables, lens=np.append(self.lens, U32(0)), starts=self.starts, parents=self.parents,
                                      drafts=self.drafts, targets=self.targets if logits is None else np.full_like(self.targets, 0xAAAAAAAA),
                                      lens_out=np.full(B + 1, 0xBBBBBBBB, U32), counts=np.full(B + 1, 0xBBBBBBBB, U32),
                                      tokens=np.full(self.rows + 1, 0xBBBBBBBB, U32), stack=self.stack,
                                      count=np.array([self.count], U32), count_out=np.array([0xBBBBBBBB], U32)).items()}
        batch = arc.PagedBatch(B, self.rows, self.max_pages, 0, d["tables"], d["lens"], d["starts"])
        ws = arc.DeviceBuffer(arc.tree_commit_workspace_bytes(batch))
        ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
        out = d["lens"] if in_place else d["lens_out"]
        count_out = d["count"] if in_place else d["count_out"]
        kw = dict(free_pages=d["stack"], num_pages=self.pool if num_pages is None else num_pages, free_count=d["count"],
                  free_count_out=count_out) if free_list else {}
        if logits is not None:
            dl = D(logits)
            kw.update(logits=dl.ptr + self.offset, logits_dtype=dtype, ldl=ldl, vocab=self.vocab)
        arc.tree_commit(layers, batch, arc.Tree(d["parents"], None, self.words), d["drafts"], d["targets"], out, d["counts"],
                        d["tokens"], ws, stream=stream, **kw)
        if stream is not None:
            stream.synchronize()
        return dict(counts=d["counts"].download(U32, B), tokens=d["tokens"].download(U32), lens=out.download(U32, B),
                    stack=d["stack"].download(U32), count=int(count_out.download(U32)[0]), targets=d["targets"].download(U32),
                    kv=self.dkv.download(np.uint16).reshape(self.kv.shape))

    offset = 0

    def check(self, got, free_list=True, num_pages=None):
        pools = [tuple(t[:, : self.page * self.kvd].reshape(self.pool, self.page, self.kvd) for t in layer) for layer in self.kv]
        want = tl.commit(self.shapes, self.words, self.lens, self.starts, self.tables, self.page, self.drafts[: self.rows], self.targets,
                         pools, self.stack, self.count, (self.pool if num_pages is None else num_pages) if free_list else 0)
        assert got["counts"].tolist() == want["counts"].tolist() and got["lens"].tolist() == want["lens"].tolist()
        assert np.array_equal(got["tokens"][: self.used], want["tokens"][: self.used])
        assert np.all(got["tokens"][self.used:] == 0xBBBBBBBB)
        if free_list:
            assert got["count"] == want["count"] and np.array_equal(got["stack"], want["stack"])
        whole = self.kv.copy()
        for i, (k, v) in enumerate(want["pools"]):
            whole[i, 0, :, : self.page * self.kvd] = k.reshape(self.pool, -1)
            whole[i, 1, :, : self.page * self.kvd] = v.reshape(self.pool, -1)
        assert np.array_equal(got["kv"], whole)
        return want


def trees(rng, sizes):
    return [tl.random_tree(rng, n) for n in sizes]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", ["one", "single rows", "mixed", "chain", "none agree", "all agree", "page 1", "large", "wide heads", "layers",
                                  "strides", "no requests", "many"])
def test_commit(name, in_place):
    rng = rng_of(20)
    kw = dict()
    if name == "one":
        old, shapes = [501], trees(rng, [26])
    elif name == "single rows":
        old, shapes = [0, 15, 16], trees(rng, [1, 1, 1])
    elif name == "mixed":
        old, shapes, kw = [40, 0, 7, 100, 31], [tl.random_tree(rng, 20), 50, [], tl.chain(1), tl.random_tree(rng, 32)], dict(words=1, rows=4)
    elif name == "chain":
        old, shapes, kw = [5, 17], [tl.chain(40), tl.chain(33)], dict(agree=0.95)
    elif name == "none agree":
        old, shapes, kw = [30, 64], trees(rng, [30, 40]), dict(agree=0.0, vocab=100000)
    elif name == "all agree":
        old, shapes, kw = [30, 0, 90], [tl.chain(64), tl.star(20), tl.random_tree(rng, 50)], dict(agree=1.0)
    elif name == "page 1":
        old, shapes, kw = [3, 0], trees(rng, [20, 9]), dict(page=1)
    elif name == "large":
        old, shapes, kw = [100], [tl.random_tree(rng, 1024)], dict(words=32, agree=0.95, vocab=3)
    elif name == "wide heads":
        old, shapes, kw = [20], trees(rng, [30]), dict(kv_heads=40, dim=128, layers=1, dtype=arc.BF16)
    elif name == "layers":
        old, shapes, kw = [20, 9], trees(rng, [30, 12]), dict(layers=64, kv_heads=1)
    elif name == "strides":
        old, shapes, kw = [20, 9], trees(rng, [30, 12]), dict(stride_pad=24, page=32)
    elif name == "no requests":
        old, shapes = [], []
    else:
        n = 700
        old = rng.integers(0, 60, n).tolist()
        shapes = [tl.random_tree(rng, int(x)) if x else [] for x in rng.integers(0, 30, n)]
        kw = dict(page=4, kv_heads=1, layers=1)
    run = CommitRun(old, shapes, seed=21, **kw)
    run.check(run.run(in_place=in_place))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", ["chunk", "empty", "single row", "chain", "page 1", "wide heads", "layers", "strides", "rows behind", "without room", "no list"])
def test_commit_of_one_request(name, in_place):
    rng = rng_of(30)
    kw = dict(chunk=dict(words=1), chain=dict(agree=0.97), layers=dict(layers=64), strides=dict(stride_pad=24, page=32), empty=dict(rows=3))
    kw["page 1"], kw["wide heads"], kw["rows behind"] = dict(page=1), dict(kv_heads=40, dim=128, layers=3, dtype=arc.BF16), dict(rows=9)
    kw["without room"] = kw["no list"] = dict(agree=0.1, page=4)
    shape = dict(chunk=70, empty=[], chain=tl.chain(200)).get(name, tl.chain(1) if name == "single row" else tl.random_tree(rng, 60))
    run = CommitRun([37], [shape], seed=31, **kw.get(name, {}))
    if name == "no list":
        run.check(run.run(in_place=in_place, free_list=False), free_list=False)
    elif name == "without room":
        run.check(run.run(in_place=in_place, num_pages=run.count + 5), num_pages=run.count + 5)
    else:
        run.check(run.run(in_place=in_place))


def test_commit_of_one_request_from_logits():
    run = CommitRun([37], [tl.random_tree(rng_of(32), 60)], seed=32, vocab=1003, agree=0.8)
    logits = rng_of(33).standard_normal((run.rows, 1003)).astype(np.float32)
    logits[np.arange(run.rows), run.targets[: run.rows]] = 50.0
    got = run.run(logits=logits, ldl=1003)
    assert np.array_equal(got["targets"][: run.rows], run.targets[: run.rows])
    run.check(got)


def test_commit_without_a_free_list():
    run = CommitRun([20, 9], trees(rng_of(22), [30, 12]), seed=22)
    got = run.run(free_list=False)
    run.check(got, free_list=False)
    assert got["count"] == 0xBBBBBBBB and np.array_equal(got["stack"], run.stack)


def test_commit_free_list_without_room():
    run = CommitRun([20, 9, 40], trees(rng_of(23), [60, 50, 64]), seed=23, agree=0.1, page=4)
    room = run.count + 5
    run.check(run.run(num_pages=room), num_pages=room)


def test_commit_leaves_rows_whose_page_is_none():
    run = CommitRun([12, 3], [tl.chain(20), tl.chain(20)], seed=24, agree=1.0, page=4)
    shapes = run.shapes
    run.shapes = [[tl.NONE, 0, 0] + list(range(2, 19)), shapes[1]]  # the way leaves node 1 out: every node moves
    run.parents[:20] = run.shapes[0]
    run.drafts[1] = run.targets[0] + 1
    run.drafts[2] = run.targets[0]
    run.tables[0, 5] = run.pool + 7
    run.check(run.run(free_list=False), free_list=False)


def test_commit_takes_the_first_of_equal_children():
    run = CommitRun([10], [[tl.NONE, 0, 0, 0, 1, 2, 3]], seed=25)
    run.drafts[:7] = [0, 4, 4, 4, 5, 5, 5]
    run.targets[:7] = [4, 9, 5, 5, 6, 7, 8]
    want = run.check(run.run())
    assert want["counts"][0] == 2 and want["tokens"][:3].tolist() == [4, 9, arc.NO_TOKEN]


@pytest.mark.parametrize("dtype", [arc.F32, arc.F16, arc.BF16])
@pytest.mark.parametrize("vocab,pad,shift", [(1, 0, 0), (3, 2, 1), (7, 0, 1), (255, 1, 0), (1000, 24, 3), (1003, 0, 1), (152064, 0, 0), (40001, 7, 5)])
def test_commit_from_logits(vocab, pad, shift, dtype):
    rng = rng_of(vocab, dtype)
    run = CommitRun([20, 9], [tl.random_tree(rng, 12), tl.random_tree(rng, 5)], seed=26, rows=2, vocab=vocab)
    ldl = vocab + pad
    x = (rng.integers(-9, 9, (run.rows, ldl)) if vocab < 2000 else rng.standard_normal((run.rows, ldl)) * 3).astype(np.float32)
    x[0, :vocab] = -np.inf
    x[1, : vocab // 2] = np.nan
    x[2, :vocab] = np.nan
    x[3, vocab - 1] = np.inf
    x[4, :vocab] = -7.0  # all equal
    x[:, vocab:] = 1e4  # not a part of the row
    # what the target says, agreed to by most drafts
    bits = x if dtype == arc.F32 else pl.to_bits(x, dtype)
    vals = x if dtype == arc.F32 else pl.from_bits(bits, dtype)
    said = [tl.argmax(r[:vocab]) if vocab < 3000 else int(np.nanargmax(np.where(np.isnan(r[:vocab]), -np.inf, r[:vocab]))) for r in vals]
    said[2] = 0
    run.targets[: run.rows] = said
    for b, s in enumerate(run.shapes):
        for i in range(1, len(s)):
            run.drafts[run.starts[b] + i] = run.targets[run.starts[b] + s[i]] if rng.random() < 0.8 else vocab + 5
    # rows that start `shift` elements behind a 16-byte border, in an allocation that ends with the last one
    flat = np.concatenate([np.zeros(shift, bits.dtype), bits.reshape(-1)[: (run.rows - 1) * ldl + vocab]])
    run.offset = shift * bits.itemsize
    got = run.run(logits=flat, ldl=ldl, dtype=dtype)
    assert got["targets"][: run.used].tolist() == said[: run.used]
    assert np.all(got["targets"][run.used:] == 0xAAAAAAAA)
    run.check(got)


def test_commit_from_many_logits():
    run = CommitRun([5] * 200, [tl.chain(16)] * 200, seed=27, kv_heads=1, layers=1, vocab=300)
    x = rng_of(28).standard_normal((run.rows, 300)).astype(np.float32)
    run.targets[: run.rows] = x.argmax(1)
    for b in range(200):
        for i in range(1, 16):
            if rng_of(b, i).random() < 0.8:
                run.drafts[16 * b + i] = run.targets[16 * b + i - 1]
    got = run.run(logits=x, ldl=300)
    assert np.array_equal(got["targets"][: run.rows], run.targets[: run.rows])
    run.check(got)


def test_commits_on_their_own_streams():
    runs = [CommitRun([60 + i, 5], trees(rng_of(30 + i), [40, 30]), seed=40 + i) for i in range(3)]
    streams = [arc.Stream() for _ in runs]
    for r, s in zip(runs, streams):
        r.check(r.run(stream=s))
