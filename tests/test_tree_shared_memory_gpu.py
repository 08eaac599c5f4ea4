"""The end of a draft-tree step over pools whose pages lie in turns in one buffer, with a small array in the room behind
each page: nothing is shared, so the call takes it."""
import numpy as np
import pytest

import arcllm_amd as arc
import tree_lib as tl
from test_tree_gpu import U32, CommitRun, D, rng_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


class InTurns(CommitRun):
    """A page's bytes of all layers' K and V side by side, then 128 bytes of room."""

    def run(self):
        B, (kv_heads, dim, dt), page = len(self.shapes), self.dims, self.page * self.kvd
        order = np.ascontiguousarray(self.kv.transpose(2, 0, 1, 3))  # [pool][layers][2][page]
        room = np.full((self.pool, 64), 0xBBBB, np.uint16)
        buf = D(np.concatenate([order.reshape(self.pool, -1), room], 1))
        stride = 2 * self.layers * page + 64
        at = lambda p, n: buf.ptr + 2 * (p * stride + n * page)  # noqa: E731
        layers = [arc.KvPages(at(0, 2 * i), at(0, 2 * i + 1), self.pool, self.page, kv_heads, dim, dt, stride) for i in range(self.layers)]
        d = {k: D(v) for k, v in dict(tables=self.tables, lens=self.lens, starts=self.starts, parents=self.parents, drafts=self.drafts,
                                      targets=self.targets, tokens=np.full(self.rows + 1, 0xBBBBBBBB, U32), stack=self.stack,
                                      count=np.array([self.count], U32)).items()}
        # counts, lens_out and free_count_out behind pages 0, 1 and 2
        counts, lens_out, count_out = (at(p, 2 * self.layers) for p in range(3))
        batch = arc.PagedBatch(B, self.rows, self.max_pages, 0, d["tables"], d["lens"], d["starts"])
        ws = arc.DeviceBuffer(arc.tree_commit_workspace_bytes(batch))
        arc.tree_commit(layers, batch, arc.Tree(d["parents"], None, self.words), d["drafts"], d["targets"], lens_out, counts, d["tokens"], ws,
                        free_pages=d["stack"], num_pages=self.pool, free_count=d["count"], free_count_out=count_out)
        out = buf.download(np.uint16).reshape(self.pool, stride)
        said = [np.ascontiguousarray(out[p, -64:]).view(U32) for p in range(3)]
        used = (B, B, 1)
        for p in range(self.pool):
            behind = used[p] if p < 3 else 0
            assert np.all(out[p, 2 * self.layers * page + 2 * behind:] == 0xBBBB)
        kv = np.ascontiguousarray(out[:, :-64].reshape(self.pool, self.layers, 2, page).transpose(1, 2, 0, 3))
        return dict(counts=said[0][:B], lens=said[1][:B], count=int(said[2][0]), tokens=d["tokens"].download(U32), stack=d["stack"].download(U32), kv=kv)


@pytest.mark.parametrize("sizes,layers,page", [([40], 3, 4), ([26], 28, 16), ([30, 1, 55], 2, 8), ([64] * 20, 64, 4)])
def test_pages_in_turns(sizes, layers, page):
    rng = rng_of(60, len(sizes), layers)
    run = InTurns([int(x) for x in rng.integers(0, 50, len(sizes))], [tl.random_tree(rng, n) for n in sizes], page=page, layers=layers, kv_heads=1, seed=61)
    run.check(run.run())
