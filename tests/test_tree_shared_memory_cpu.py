"""The end of a draft-tree step refuses pools that lie over each other and arrays that lie in a pool or in the logits,
before any launch."""
import pytest

import arcllm_amd as arc

A = 0x1000000  # addresses that are never followed
PAGE = 16 * 2 * 128 * 2  # bytes of a page: 16 positions of 2 heads of 128


def pages(k, v, n=8, stride=None):
    return arc.KvPages(k, v, n, 16, 2, 128, arc.F16, stride)


def commit(layers=None, **over):
    kw = dict(tables=A, lens=2 * A, starts=3 * A, parents=4 * A, drafts=5 * A, targets=6 * A, lens_out=7 * A, counts=8 * A, tokens=9 * A,
              workspace=10 * A, free_pages=11 * A, free_count=12 * A, free_count_out=13 * A, logits=None, ldl=100)
    kw.update(over)
    batch = arc.PagedBatch(2, 6, 4, 4, kw["tables"], kw["lens"], kw["starts"])
    more = dict(logits=kw["logits"], logits_dtype=arc.F32, ldl=kw["ldl"], vocab=100) if kw["logits"] else {}
    arc.tree_commit(layers or [pages(40 * A, 41 * A), pages(42 * A, 43 * A)], batch, arc.Tree(kw["parents"], None, 1), kw["drafts"], kw["targets"],
                    kw["lens_out"], kw["counts"], kw["tokens"], kw["workspace"], free_pages=kw["free_pages"], num_pages=8,
                    free_count=kw["free_count"], free_count_out=kw["free_count_out"], **more)


def refused(fn):
    with pytest.raises(arc.ArcError, match="shares? memory|twice") as e:
        fn()
    assert e.value.code == 1


@pytest.mark.parametrize("layers", [
    [pages(40 * A, 40 * A + 8 * PAGE - 16)],                                     # V begins in K's last page
    [pages(40 * A, 41 * A), pages(41 * A + PAGE, 43 * A)],
    [pages(40 * A, 41 * A), pages(42 * A, 39 * A), pages(50 * A, 42 * A - 16)],
    [pages(40 * A, 40 * A + PAGE - 16, stride=2 * PAGE // 2)],                   # two pools in turns, a page and less from one to the next
    [pages(40 * A, 40 * A + PAGE, stride=PAGE // 2 + 8)],
    [pages(40 * A, 40 * A + PAGE, stride=PAGE), pages(40 * A + 2 * PAGE - 16, 60 * A, stride=PAGE)],
    [pages(40 * A, 40 * A + PAGE - 16, n=1, stride=5 * PAGE)],
], ids=range(7))
def test_pools_over_each_other(layers):
    refused(lambda: commit(layers))


ARRAYS = ["tables", "lens", "starts", "parents", "drafts", "targets", "lens_out", "counts", "tokens", "workspace", "free_pages", "free_count",
          "free_count_out"]


@pytest.mark.parametrize("name", ARRAYS)
def test_arrays_in_a_pool(name):
    for at in (40 * A, 41 * A + 8 * PAGE - 256, 43 * A + 3 * PAGE):
        refused(lambda: commit(**{name: at}))


@pytest.mark.parametrize("name", ["lens_out", "free_count_out", "counts", "tables", "workspace"])
def test_arrays_in_a_pool_whose_pages_lie_apart(name):
    # K and V in turns, a page of room behind each V: the room is free, a page's last bytes are not
    layers = [pages(40 * A, 40 * A + PAGE, stride=3 * PAGE // 2)]
    refused(lambda: commit(layers, **{name: 40 * A + 2 * PAGE - 256}))
    refused(lambda: commit(layers, **{name: 40 * A + 5 * 3 * PAGE + PAGE}))


@pytest.mark.parametrize("name", ["targets", "lens_out", "counts", "tokens", "workspace", "free_pages", "free_count_out"])
def test_what_is_written_in_the_logits(name):
    refused(lambda: commit(logits=20 * A, **{name: 20 * A}))
    refused(lambda: commit(logits=20 * A, ldl=256, **{name: 20 * A + 1024 * 5 + 256}))


def test_logits_in_a_pool():
    refused(lambda: commit(logits=40 * A))
    refused(lambda: commit(logits=42 * A - 1024 * 5 - 16, ldl=256))
