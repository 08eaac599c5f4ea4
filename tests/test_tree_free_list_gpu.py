"""The pages that a draft-tree step's end returns, where the table has entries that are no page of the pool: those
stay off the free list, all others go onto it in order."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_lib as pl
import tree_lib as tl
from test_tree_gpu import CommitRun, rng_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


def returned(run, lens):
    """The pages behind lens that each tree held, requests in order, without those that are none."""
    out = []
    for b, shape in enumerate(run.shapes):
        if isinstance(shape, int):
            continue
        for p in range(pl.pages_of(int(lens[b]), run.page), pl.pages_of(int(run.lens[b]), run.page)):
            if run.tables[b, p] < run.pool:
                out.append(int(run.tables[b, p]))
    return out


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("sizes,page,bad", [([60], 4, 0.3), ([60], 4, 1.0), ([1000], 1, 0.4), ([300], 1, 0.0), ([60, 1, 45], 4, 0.3), ([33] * 300, 2, 0.5),
                                            ([20, 50, 30], 1, 1.0)])
def test_entries_that_are_no_page_stay_off_the_list(sizes, page, bad, in_place):
    rng = rng_of(50, len(sizes), page)
    old = [int(x) for x in rng.integers(0, 40, len(sizes))]
    run = CommitRun(old, [tl.random_tree(rng, n) for n in sizes], page=page, seed=51, kv_heads=1, layers=2, agree=0.5)
    # of each request's own pages behind its context, some are none: the pool's end, one behind it, far out
    for b, n in enumerate(sizes):
        for p in range(pl.pages_of(old[b], page), pl.pages_of(int(run.lens[b]), page)):
            if rng.random() < bad:
                run.tables[b, p] = (run.pool, run.pool + 1, 0xFFFFFFFF)[int(rng.integers(3))]
    got = run.run(in_place=in_place)
    run.check(dict(got, stack=None), free_list=False)
    back = returned(run, got["lens"])
    assert got["count"] == run.count + len(back)
    assert got["stack"][: run.count].tolist() == run.stack[: run.count].tolist()
    assert got["stack"][run.count: run.count + len(back)].tolist() == back
    assert np.all(got["stack"][run.count + len(back):] == 0xEEEEEEEE)
    if bad == 1.0:
        assert not back


@pytest.mark.parametrize("sizes", [[600], [90, 70]])
def test_a_list_without_room_keeps_the_first(sizes):
    rng = rng_of(52, len(sizes))
    run = CommitRun([7] * len(sizes), [tl.random_tree(rng, n) for n in sizes], page=1, seed=53, kv_heads=1, layers=1, agree=0.1)
    for b, n in enumerate(sizes):
        run.tables[b, 10: 7 + n: 3] = 0xFFFFFFF0
    room = run.count + 9
    got = run.run(num_pages=room)
    run.check(dict(got, stack=None), free_list=False)
    back = returned(run, got["lens"])[:9]
    assert len(back) == 9 and got["count"] == room
    assert got["stack"][run.count: room].tolist() == back and np.all(got["stack"][room:] == 0xEEEEEEEE)
