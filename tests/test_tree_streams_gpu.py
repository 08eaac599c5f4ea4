"""Draft-tree calls under way on several streams at once, each with its own workspace: everything is launched, several times,
before anything is waited for."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_lib as pl
import tree_lib as tl
from test_tree_gpu import U32, CommitRun, D, rng_of

pytestmark = pytest.mark.gpu

TIMES = 3


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


class Commits(CommitRun):
    """TIMES calls on buffers of their own, which share the workspace, as calls of one stream may."""

    def prepare(self, logits):
        B, (kv_heads, dim, dt), size = len(self.shapes), self.dims, self.kv[0, 0].nbytes
        self.x = None
        if logits:
            self.x = rng_of(70).standard_normal((self.rows, self.vocab)).astype(np.float32)
            self.x[np.arange(self.rows), self.targets[: self.rows]] = 50.0
        self.calls = []
        for _ in range(TIMES):
            kv = D(self.kv)
            layers = [arc.KvPages(kv.ptr + 2 * i * size, kv.ptr + (2 * i + 1) * size, self.pool, self.page, kv_heads, dim, dt) for i in range(self.layers)]
            d = {k: D(v) for k, v in dict(tables=self.tables, lens=self.lens, starts=self.starts, parents=self.parents, drafts=self.drafts,
                                          targets=np.full_like(self.targets, 0xAAAAAAAA) if logits else self.targets,
                                          lens_out=np.full(B, 0xBBBBBBBB, U32), counts=np.full(B, 0xBBBBBBBB, U32),
                                          tokens=np.full(self.rows + 1, 0xBBBBBBBB, U32), stack=self.stack, count=np.array([self.count], U32),
                                          count_out=np.array([0xBBBBBBBB], U32)).items()}
            if logits:
                d["logits"] = D(self.x)
            self.calls.append((kv, layers, d, arc.PagedBatch(B, self.rows, self.max_pages, 0, d["tables"], d["lens"], d["starts"])))
        self.ws = arc.DeviceBuffer(arc.tree_commit_workspace_bytes(self.calls[0][3]))
        self.ws.upload(np.full(self.ws.nbytes, 0xFF, np.uint8))

    def launch(self, i, stream):
        _, layers, d, batch = self.calls[i]
        more = dict(logits=d["logits"], logits_dtype=arc.F32, ldl=self.vocab, vocab=self.vocab) if self.x is not None else {}
        arc.tree_commit(layers, batch, arc.Tree(d["parents"], None, self.words), d["drafts"], d["targets"], d["lens_out"], d["counts"], d["tokens"],
                        self.ws, free_pages=d["stack"], num_pages=self.pool, free_count=d["count"], free_count_out=d["count_out"], stream=stream,
                        **more)

    def results(self):
        for kv, _, d, _ in self.calls:
            yield dict(counts=d["counts"].download(U32), tokens=d["tokens"].download(U32), lens=d["lens_out"].download(U32),
                       stack=d["stack"].download(U32), count=int(d["count_out"].download(U32)[0]), kv=kv.download(np.uint16).reshape(self.kv.shape))


def run_together(jobs):
    streams = [arc.Stream() for _ in jobs]
    arc.synchronize()
    for i in range(TIMES):
        for job, s in zip(jobs, streams):
            job.launch(i, s)
    for s in streams:
        s.synchronize()


@pytest.mark.parametrize("logits", [False, True])
def test_commits(logits):
    jobs = []
    for n, (old, sizes) in enumerate([([60, 5], [40, 30]), ([501], [26]), ([9] * 30, [20] * 30), ([33], [200])]):
        rng = rng_of(71, n)
        jobs.append(Commits(old, [tl.random_tree(rng, m) for m in sizes], seed=72 + n, layers=4, vocab=9001 if logits else 50, agree=0.8))
        jobs[-1].prepare(logits)
    run_together(jobs)
    for job in jobs:
        for got in job.results():
            job.check(got)


class Attention:
    def __init__(self, old, shapes, heads, dim, seed, **kw):
        self.s = tl.TreeStep(old, shapes, 16, *heads, dim, arc.F16, seed).upload()
        self.kw = kw
        self.outs = [D(np.full((self.s.rows, self.s.ldo), 0xABCD, np.uint16)) for _ in range(TIMES)]
        self.ws = arc.DeviceBuffer(arc.tree_attention_workspace_bytes(self.s.pages, self.s.batch, self.s.hpk))
        self.ws.upload(np.full(self.ws.nbytes, 0xFF, np.uint8))

    def launch(self, i, stream):
        s = self.s
        arc.tree_attention(s.pages, s.batch, s.tree, s.dq, s.ldq, s.hpk, self.outs[i], s.ldo, self.ws, stream=stream, **self.kw)


def test_attention():
    rng = rng_of(73)
    tree = lambda n: tl.random_tree(rng, n)  # noqa: E731
    jobs = [Attention([3000, 200], [tree(40), tree(9)], (4, 7), 128, 1), Attention([30] * 20, [tree(3) for _ in range(20)], (2, 4), 64, 2),
            Attention([700], [tree(100)], (2, 8), 128, 3, window=300, sinks=4), Attention([90, 10], [tl.chain(1), tl.chain(1)], (2, 4), 128, 4)]
    run_together(jobs)
    for job in jobs:
        bits = [out.download(np.uint16).reshape(-1, job.s.ldo) for out in job.outs]
        job.s.check(bits[0], **job.kw)
        assert all(np.array_equal(bits[0], b) for b in bits[1:])


def test_plans():
    jobs = []
    for n in range(3):
        rng = rng_of(74, n)
        s = tl.TreeStep([5 + n] * 40, [tl.random_tree(rng, 20 + n) for _ in range(40)], 16, 1, 1, 64, arc.F16, n).upload()
        s.outs = [(D(np.full((s.rows, s.words), 7, U32)), D(np.full(s.rows, 7, U32))) for _ in range(TIMES)]

        def launch(i, stream, s=s):
            masks, positions = s.outs[i]
            batch = arc.PagedBatch(len(s.old), s.rows, s.max_pages, s.max_new, s.dtables, s.dlens, s.dstarts, positions)
            arc.tree_plan(batch, arc.Tree(s.dparents, masks, s.words), stream=stream)

        s.launch = launch
        jobs.append(s)
    run_together(jobs)
    for s in jobs:
        want = tl.plan(s.shapes, s.words, s.rows, [int(x) for x in s.lens], np.zeros((s.rows, s.words), U32), np.zeros(s.rows, U32))
        for masks, positions in s.outs:
            assert np.array_equal(masks.download(U32).reshape(s.rows, -1), want[0]) and np.array_equal(positions.download(U32), want[1])
