"""The draft-tree entry points without a GPU: every refusal comes before any launch, and the oracle's own
statements on hand-written trees."""
import ctypes as C

import numpy as np
import pytest

import arcllm_amd as arc
import tree_lib as tl

A = 0x10000  # an address that is never followed: every call here is refused first


def pages(**over):
    d = dict(k=A, v=2 * A, num_pages=8, page_size=16, kv_heads=2, head_dim=128, dtype=arc.F16)
    d.update(over)
    return arc.KvPages(**d)


def batch(**over):
    d = dict(requests=2, tokens=4, max_pages=4, max_new=4, tables=A, lens=A, starts=A, positions=A, slots=A)
    d.update(over)
    return arc.PagedBatch(**d)


def tree(**over):
    d = dict(parents=A, masks=A, mask_words=1)
    d.update(over)
    return arc.Tree(**d)


def refused(fn):
    with pytest.raises(arc.ArcError) as e:
        fn()
    assert e.value.code in (1, 2) and len(str(e.value)) > 20


BIG = 33


@pytest.mark.parametrize("call", [
    lambda: arc.tree_plan(batch(requests=(1 << 20) + 1), tree()), lambda: arc.tree_plan(batch(tokens=(1 << 24) + 1), tree()),
    lambda: arc.tree_plan(batch(lens=None), tree()), lambda: arc.tree_plan(batch(starts=None), tree()),
    lambda: arc.tree_plan(batch(positions=None), tree()), lambda: arc.tree_plan(batch(), tree(parents=None)),
    lambda: arc.tree_plan(batch(), tree(masks=None)), lambda: arc.tree_plan(batch(), tree(mask_words=0)),
    lambda: arc.tree_plan(batch(), tree(mask_words=BIG)),
])
def test_plan_refusals(call):
    refused(call)


def test_plan_of_nothing_is_done():
    arc.tree_plan(batch(requests=0), tree())
    arc.tree_plan(batch(tokens=0), tree())


def attention(p=None, b=None, t=None, q=A, ldq=512, hpk=2, out=8 * A, ldo=512, ws=4 * A, **kw):
    arc.tree_attention(p or pages(), b or batch(), t or tree(), q, ldq, hpk, out, ldo, ws, **kw)


@pytest.mark.parametrize("call", [
    lambda: attention(t=tree(masks=None)), lambda: attention(t=tree(mask_words=0)), lambda: attention(t=tree(mask_words=BIG)),
    lambda: attention(b=batch(positions=None), window=5), lambda: attention(b=batch(tables=None)), lambda: attention(b=batch(max_pages=0)),
    lambda: attention(p=pages(head_dim=96)), lambda: attention(p=pages(dtype=arc.F32)), lambda: attention(q=None),
    lambda: attention(out=A), lambda: attention(ws=4 * A + 64), lambda: attention(ldq=504), lambda: attention(hpk=0),
    lambda: attention(scale=float("inf")), lambda: attention(b=batch(tokens=(1 << 24) + 1)),
])
def test_attention_refusals(call):
    refused(call)


def test_attention_of_nothing_is_done():
    attention(b=batch(tokens=0))
    attention(b=batch(requests=0, positions=None))
    attention(b=batch(tokens=0), t=tree(parents=None))  # attention reads masks only


def commit(layers=None, b=None, t=None, drafts=A, targets=A, lens_out=A, counts=A, tokens=A, ws=4 * A, **kw):
    arc.tree_commit([pages()] if layers is None else layers, b or batch(), t or tree(), drafts, targets, lens_out, counts, tokens, ws, **kw)


LIST = dict(free_pages=A, num_pages=8, free_count=A, free_count_out=A)
LOGITS = dict(logits=A, logits_dtype=arc.F32, ldl=100, vocab=100)


@pytest.mark.parametrize("call", [
    lambda: commit(layers=[]), lambda: commit(layers=[pages()] * 65), lambda: commit(layers=[pages(), pages(kv_heads=1)]),
    lambda: commit(layers=[pages(), pages(num_pages=9)]), lambda: commit(layers=[pages(), pages(page_stride=16 * 256 + 8)]),
    lambda: commit(layers=[pages(k=None)]), lambda: commit(b=batch(tables=None)), lambda: commit(b=batch(lens=None)),
    lambda: commit(t=tree(parents=None)), lambda: commit(t=tree(mask_words=BIG)), lambda: commit(drafts=None),
    lambda: commit(targets=None), lambda: commit(lens_out=None), lambda: commit(counts=None), lambda: commit(tokens=None),
    lambda: commit(ws=None), lambda: commit(ws=4 * A + 4), lambda: commit(**{**LIST, "free_count": None}),
    lambda: commit(**{**LIST, "free_count_out": None}), lambda: commit(**{**LIST, "num_pages": 0}),
    lambda: commit(**{**LOGITS, "vocab": 0}), lambda: commit(**{**LOGITS, "ldl": 99}), lambda: commit(**{**LOGITS, "logits_dtype": 7}),
    lambda: commit(**{**LOGITS, "logits": A + 2}), lambda: commit(**{**LOGITS, "vocab": (1 << 24) + 1, "ldl": 1 << 25}),
    lambda: commit(b=batch(tokens=(1 << 20) + 1), **LOGITS),
])
def test_commit_refusals(call):
    refused(call)


def apart(**over):
    """A commit whose arrays lie apart, but for `over`; none of them is followed."""
    kw = dict(layers=[pages(k=(40 + 2 * i) * A, v=(41 + 2 * i) * A) for i in range(3)],
              b=batch(tables=A, lens=2 * A, starts=3 * A), t=tree(parents=4 * A), drafts=5 * A, targets=6 * A, lens_out=7 * A, counts=8 * A,
              tokens=9 * A, ws=10 * A, free_pages=11 * A, num_pages=8, free_count=12 * A, free_count_out=13 * A)
    commit(**{**kw, **over})


@pytest.mark.parametrize("over", [
    dict(layers=[pages(), pages(k=3 * A, v=4 * A), pages()]), dict(layers=[pages(k=A, v=A)]), dict(layers=[pages(), pages(k=2 * A, v=3 * A)]),
    dict(tokens=6 * A), dict(tokens=5 * A + 4), dict(tokens=8 * A), dict(counts=7 * A), dict(counts=2 * A), dict(lens_out=2 * A + 4),
    dict(lens_out=3 * A), dict(lens_out=4 * A + 12), dict(free_pages=A), dict(free_count_out=12 * A - 2), dict(free_count_out=11 * A + 28),
    dict(ws=9 * A), dict(free_pages=10 * A + 256), dict(targets=5 * A, **LOGITS), dict(targets=9 * A, **LOGITS),
], ids=str)
def test_commit_of_shared_memory_is_refused(over):
    with pytest.raises(arc.ArcError, match="twice|shares memory"):
        apart(**over)


def test_plan_of_shared_memory_is_refused():
    b = batch(lens=2 * A, starts=3 * A, positions=4 * A)
    for t in (tree(parents=5 * A, masks=4 * A), tree(parents=5 * A, masks=5 * A + 12), tree(parents=4 * A, masks=6 * A),
              tree(parents=5 * A, masks=2 * A), tree(parents=5 * A, masks=3 * A - 4, mask_words=1)):
        with pytest.raises(arc.ArcError, match="share memory"):
            arc.tree_plan(b, t)


def test_commit_takes_pages_only():
    with pytest.raises(TypeError):
        commit(layers=[pages(), 5])


def test_null_structs():
    L = arc.lib()
    p, b, t = pages(), batch(), tree()
    assert L.arc_tree_plan(None, C.byref(t), None) == 1 and L.arc_tree_plan(C.byref(b), None, None) == 1
    assert L.arc_tree_attention(C.byref(p), C.byref(b), None, A, 512, 2, 0.0, 0, 0, 8 * A, 512, 4 * A, None) == 1
    assert L.arc_tree_attention_workspace_bytes(None, C.byref(b), 2) == 0
    assert L.arc_tree_commit_workspace_bytes(None) == 0
    assert L.arc_tree_commit(None, 1, C.byref(b), C.byref(t), 0, None, 0, 0, A, A, A, A, A, None, 0, None, None, A, None) == 1


def test_workspaces_grow_with_the_step():
    small, large = (arc.tree_commit_workspace_bytes(batch(tokens=n, requests=3)) for n in (1, 4000))
    assert 0 < small < large
    assert arc.tree_attention_workspace_bytes(pages(), batch(), 2) == arc.paged_attention_workspace_bytes(pages(), batch(), 2)


# ------------------------------------------------------- the oracle's statements
def test_oracle_masks_and_walk():
    #      0 -> 1 -> 3, 0 -> 2 -> 4 -> 5
    parents = [tl.NONE, 0, 0, 1, 2, 4]
    assert [sorted(tl.ancestors(parents, i)) for i in range(6)] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 4, 5]]
    masks, pos = tl.plan([parents], 1, 6, [16], np.zeros((6, 1), np.uint32), np.zeros(6, np.uint32))
    assert masks[:, 0].tolist() == [1, 3, 5, 11, 21, 53] and pos.tolist() == [10, 11, 11, 12, 12, 13]
    drafts = [9, 7, 8, 1, 2, 3]
    assert tl.walk(parents, drafts, [8, 0, 2, 0, 3, 6]) == [0, 2, 4, 5]
    assert tl.walk(parents, drafts, [7, 5, 2, 0, 3, 6]) == [0, 1]
    assert tl.walk(parents, drafts, [1, 1, 1, 1, 1, 1]) == [0]
    assert tl.ancestors([tl.NONE, 1, 5, 0], 1) == [1] and tl.ancestors([tl.NONE, 1, 5, 0], 2) == [2]  # no parent before them


def test_oracle_argmax():
    nan = float("nan")
    assert [tl.argmax(r) for r in ([1, 3, 3], [nan, 2, 1], [nan, nan], [-np.inf, -np.inf], [nan, -np.inf])] == [1, 1, 0, 0, 1]
