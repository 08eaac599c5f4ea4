"""The paged-cache entry points without a GPU: every refusal comes before any launch,
the phases of rope_phases against their definition in rational arithmetic, the
oracle's own plan on hand-written steps, and the types' rounding."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

import arcllm_amd as arc
import paged_lib as pl

A = 0x10000  # an address that is never followed: every call here is refused first


def pages(**over):
    d = dict(k=A, v=2 * A, num_pages=8, page_size=16, kv_heads=2, head_dim=128, dtype=arc.F16)
    d.update(over)
    return arc.KvPages(**d)


def batch(**over):
    d = dict(requests=2, tokens=4, max_pages=4, max_new=4, tables=A, lens=A, starts=A, positions=A, slots=A)
    d.update(over)
    return arc.PagedBatch(**d)


BAD_PAGES = [dict(k=None), dict(v=None), dict(num_pages=0), dict(page_size=0), dict(page_size=12), dict(page_size=1 << 17),
             dict(kv_heads=0), dict(kv_heads=257), dict(head_dim=80), dict(head_dim=0), dict(dtype=arc.F32), dict(dtype=7),
             dict(k=A + 8), dict(v=A + 2), dict(page_stride=16 * 256 - 8), dict(page_stride=16 * 256 + 4),
             dict(num_pages=1 << 28)]


def refused(fn):
    with pytest.raises(arc.ArcError) as e:
        fn()
    assert e.value.code in (1, 2) and len(str(e.value)) > 20


def attention(p=None, b=None, q=A, ldq=512, hpk=2, out=8 * A, ldo=512, ws=4 * A, **kw):
    arc.paged_attention(p or pages(), b or batch(), q, ldq, hpk, out, ldo, ws, **kw)


@pytest.mark.parametrize("over", BAD_PAGES, ids=str)
def test_bad_pages(over):
    p = pages(**over)
    refused(lambda: attention(p))
    refused(lambda: append(p))
    refused(lambda: arc.paged_attention_workspace_bytes(p, batch(), 2))


@pytest.mark.parametrize("call", [
    lambda: attention(b=batch(tables=None)), lambda: attention(b=batch(lens=None)), lambda: attention(b=batch(starts=None)),
    lambda: attention(b=batch(max_pages=0)), lambda: attention(b=batch(max_pages=(1 << 27) + 1)),
    lambda: attention(b=batch(requests=(1 << 20) + 1)), lambda: attention(b=batch(tokens=(1 << 24) + 1)),
    lambda: attention(q=None), lambda: attention(out=None), lambda: attention(ws=None), lambda: attention(ws=4 * A + 128),
    lambda: attention(q=A + 8), lambda: attention(out=8 * A + 4), lambda: attention(ldq=504), lambda: attention(ldo=508),
    lambda: attention(ldq=516), lambda: attention(hpk=0), lambda: attention(hpk=65, ldq=1 << 15, ldo=1 << 15),
    lambda: attention(scale=float("nan")), lambda: attention(scale=float("inf")),
    lambda: attention(out=A),  # in place
    lambda: attention(out=A + 2 * 256),  # half of q's columns
    lambda: attention(q=A, ldq=1024, out=A + 2 * 256, ldo=1024),
    lambda: attention(q=A, ldq=768, out=A + 2 * 512, ldo=768),  # out's end meets the next row of q
])
def test_attention_refusals(call):
    refused(call)


def test_attention_refuses_more_work_than_its_costs_can_hold():
    # (tokens * hpk / 32 + requests) * kv_heads * hpk * (max_pages * page_size + tokens + 1024) < 2^52, also where
    # there is nothing to do, so that the sizes alone decide
    p = pages(kv_heads=256, head_dim=128, page_size=16, page_stride=16 * 256 * 128)
    width = 256 * 64 * 128
    def of(requests, max_pages):
        attention(p, batch(requests=requests, tokens=0, max_pages=max_pages), ldq=width, ldo=width, hpk=64)
    of(128, (1 << 27) - 65)  # 2^7 * 2^14 * (2^31 - 16)
    refused(lambda: of(128, (1 << 27) - 64))  # 2^52
    refused(lambda: of(1 << 20, 1 << 27))


def test_attention_of_nothing_is_done():
    attention(b=batch(tokens=0))
    attention(b=batch(requests=0))


def test_null_structs():
    L = arc.lib()
    p, b = pages(), batch()
    assert L.arc_paged_attention(None, C.byref(b), A, 512, 2, 0.0, 0, 0, 8 * A, 512, 4 * A, None) == 1
    assert L.arc_paged_attention(C.byref(p), None, A, 512, 2, 0.0, 0, 0, 8 * A, 512, 4 * A, None) == 1
    assert L.arc_paged_attention_workspace_bytes(None, C.byref(b), 2) == 0
    assert L.arc_paged_plan(None, A, A, 16, A, 8, A, A, A, None) == 1
    assert L.arc_rope_append(C.byref(p), C.byref(b), None, 0, A, 1024, None, None, None, 2, 8 * A, 512, None) == 1


# --------------------------------------------------------------------- plan
def plan(b=None, old=A, new=2 * A, page=16, free=A, num=8, count=A, count_out=A, status=A):
    arc.paged_plan(b or batch(), old, new, page, free, num, count, count_out, status)


@pytest.mark.parametrize("call", [
    lambda: plan(old=None), lambda: plan(new=None), lambda: plan(free=None), lambda: plan(count=None),
    lambda: plan(count_out=None), lambda: plan(status=None), lambda: plan(page=0), lambda: plan(page=24),
    lambda: plan(num=0), lambda: plan(num=1 << 28), lambda: plan(new=A),  # lens over new_lens
    lambda: plan(b=batch(tables=None)), lambda: plan(b=batch(positions=None)), lambda: plan(b=batch(slots=None)),
    lambda: plan(b=batch(max_pages=0)), lambda: plan(b=batch(requests=(1 << 20) + 1)),
    lambda: plan(b=batch(tokens=(1 << 24) + 1)),
])
def test_plan_refusals(call):
    refused(call)


def test_oracle_plan_by_hand():
    """Page size 4: request 0 grows over a border, 1 ends and its two pages are the next popped,
    2 is new, 3 stands still."""
    t = np.full((4, 3), 99, np.uint32)
    t[0, :1], t[1, :2], t[3, :1] = 7, (5, 6), 4
    r = pl.plan([3, 5, 0, 2], [2, arc.PAGED_RELEASE, 5, 0], 4, t, 3, 9, 5, np.array([1, 2, 3, 0, 0, 0, 0, 0], np.uint32), 3, 8)
    assert r["stack"][:5].tolist() == [1, 2, 3, 5, 6] and r["count"] == 2
    assert r["tables"].tolist() == [[7, 6, 99], [5, 6, 99], [5, 3, 99], [4, 99, 99]]
    assert r["lens"].tolist() == [5, 0, 5, 2] and r["starts"].tolist() == [0, 2, 2, 7, 7]
    assert r["positions"].tolist() == [3, 4, 0, 1, 2, 3, 4, 0, 0]
    assert r["slots"].tolist() == [31, 24, 20, 21, 22, 23, 12, arc.NO_SLOT, arc.NO_SLOT]
    assert r["status"].tolist() == [0, 0, 7, 3]


# --------------------------------------------------------------------- rope
def append(p=None, b=None, rot=128, layout=0, phases=A, xt=arc.F32, x=A, ldx=1024, hpk=2, q=64 * A, ldq=512, **kw):
    arc.rope_append(p or pages(), b or batch(), arc.Rope(phases, rot, layout), xt, x, ldx, hpk, q, ldq, **kw)


@pytest.mark.parametrize("call", [
    lambda: append(phases=None), lambda: append(phases=A + 4), lambda: append(rot=0), lambda: append(rot=12),
    lambda: append(rot=136), lambda: append(layout=2), lambda: append(xt=arc.Q4_K), lambda: append(x=None),
    lambda: append(x=A + 4), lambda: append(ldx=1016), lambda: append(ldx=1028), lambda: append(hpk=0),
    lambda: append(hpk=65, ldx=1 << 16, ldq=1 << 16), lambda: append(q=None), lambda: append(q=64 * A + 8),
    lambda: append(ldq=504), lambda: append(ldq=514), lambda: append(q_bias=A + 4), lambda: append(k_bias=A + 8),
    lambda: append(v_bias=A + 12), lambda: append(q=A), lambda: append(q=A + 4096),
    lambda: append(b=batch(slots=None)), lambda: append(b=batch(positions=None)),
    lambda: append(b=batch(tokens=(1 << 24) + 1)),
])
def test_append_refusals(call):
    refused(call)


def test_append_of_nothing_is_done():
    append(b=batch(tokens=0, positions=None, slots=None))


def test_append_may_write_q_beside_x():
    """Columns of one wide row: not shared memory, so nothing is refused for it (no rows, no launch)."""
    append(b=batch(tokens=0), x=A, ldx=2048, q=A + 4096, ldq=4096)


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=12), dict(rot=136), dict(theta=1.0), dict(theta=float("nan")),
                                dict(theta=float("inf")), dict(scaling=3), dict(scaling=1, factor=0.5),
                                dict(scaling=1, factor=float("nan")), dict(scaling=2, factor=4.0),
                                dict(scaling=2, factor=4.0, original_ctx=4096, beta_fast=1.0, beta_slow=2.0),
                                dict(scaling=2, factor=4.0, original_ctx=4096, beta_slow=-1.0),
                                dict(freq_factors=np.zeros(64)), dict(freq_factors=np.full(64, np.nan))], ids=str)
def test_phase_refusals(kw):
    kw = dict(dict(rot=128, theta=1e6), **kw)
    refused(lambda: arc.rope_phases(kw.pop("rot"), kw.pop("theta"), **kw))


@pytest.mark.parametrize("kw", [dict(), dict(scaling=arc.ROPE_LINEAR, factor=8.0),
                                dict(scaling=arc.ROPE_YARN, factor=16.0, original_ctx=8192),
                                dict(scaling=arc.ROPE_YARN, factor=40.0, original_ctx=4096, beta_fast=24.0, beta_slow=2.0),
                                dict(freq_factors=np.linspace(0.05, 9, 64, dtype=np.float32))],
                         ids=["plain", "linear", "yarn", "yarn-betas", "factors"])
@pytest.mark.parametrize("rot,theta", [(128, 1e6), (64, 1e4), (8, 500000.0)])
def test_phases(rot, theta, kw):
    """Within 2^-62 turns: the oracle's angles and the library's are computed apart, each with relative
    errors of some 2^-64 (pow, division and the blend), of values below one turn (four with factors of
    1/20); both are reduced modulo one turn exactly, pi's own error is 2^-64 relative."""
    if "freq_factors" in kw:
        kw = dict(freq_factors=kw["freq_factors"][: rot // 2])
    phases, scale = arc.rope_phases(rot, theta, **kw)
    f, want = pl.rope_freqs(rot, theta, **kw)
    assert scale == np.float32(want)
    pi2 = 2 * Fraction(31415926535897932384626433832795028841971, 10 ** 40)
    for p, x in zip(phases, f):
        hi = float(x)  # the long double as two doubles, exactly
        turns = (Fraction(hi) + Fraction(float(x - np.longdouble(hi)))) / pi2
        d = (Fraction(int(p), 2 ** 64) - turns) % 1
        assert min(d, 1 - d) <= Fraction(max(1, int(np.ceil(float(turns)))) * 4, 2 ** 64), float(x)


def test_rounding_helpers():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -3.3e38, 65504.0, 1e-7, 0.0], np.float32)
    assert pl.rounded(x[:3], arc.BF16).tolist() == [1.0, 1.0, 1 + 2.0 ** -6]
    assert np.abs(pl.rounded(x[4:6], arc.F16) - x[4:6]).max() <= 2.0 ** -25
