"""Paged entry points in forms of their own: long contexts in which no position may be lost, heads of 128 in small pages,
plans of thousands of requests and rows, q beside the rows that it comes from or beside the output."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_exact as px
import paged_lib as pl
from test_paged_gpu import PlanRun, same_plan

pytestmark = pytest.mark.gpu

SEED = 0xF0A35
D = arc.DeviceBuffer.from_array
TYPES = [arc.F16, arc.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("course", ["equal", "rising", "falling"])
@pytest.mark.parametrize("case", px.CODED, ids=str)
def test_no_position_is_lost_or_taken_twice(case, course, dtype):
    """V names the position (paged_exact.coded_rows).  An addition to an output's sum stands for 16 positions."""
    old, new, kv_heads, hpk, dim, window, sinks = case
    s = px.coded_step(old, new, kv_heads, hpk, dim, dtype, course).upload()
    bits = s.attention(window=window, sinks=sinks)
    n, rows = max(s.lens), int(s.starts[-1])
    s.check_exact(bits, dim ** -0.5, int(n) // 16, window, sinks, rows={0, 1, rows // 3, rows // 2, rows - 2, rows - 1})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("old,new,page", [([40000, 12345], [1, 1], 64), ([30000], [1], 16), ([9000, 5000], [70, 1], 32)])
def test_long_contexts_to_the_roundings(old, new, page, dtype):
    """Random values: a row within its weights' and its own rounding, scores off by (dim + 2) roundings of sum |q k|
    each, and sums of one addition for 16 positions."""
    s = px.GivenStep(old, new, page, 1, 8, 128, dtype, SEED).upload()
    bits = s.attention()
    u, scale = pl.HALF_STEP[dtype], 128 ** -0.5
    for b, row, pos in s.rows_checked({0, 1, 33, 69, 70}):
        q = pl.from_bits(s.q[row, : s.width], dtype).reshape(8, 128)
        k, v = s.K[b][: pos + 1, 0], s.V[b][: pos + 1, 0]
        ref, tol = px.exact_row(q, k, v, scale, (pos + 1) // 16, dtype)
        _, mass, off, _ = pl.attend(q, s.K[b], s.V[b], pos, scale)
        err = np.abs(pl.from_bits(bits[row, : s.width], dtype).reshape(8, 128) - ref)
        assert (err / (tol + 2 * off * (mass + np.abs(ref)))).max() <= 1.0, (b, pos)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 2, 4, 8])
@pytest.mark.parametrize("window", [0, 50])
def test_heads_of_128_in_small_pages(window, page, dtype):
    s = pl.Step([300, 11, 0, 2000], [1, 70, 5, 2], page, 2, 4, 128, dtype, SEED + page, stride_pad=24).upload()
    s.check(s.attention(window=window, sinks=3), window=window, sinks=3)


@pytest.mark.parametrize("requests", [4095, 4096, 5001])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_of_thousands_of_requests(requests, in_place):
    """The rows' launch with the starts in LDS, and without."""
    rng = np.random.default_rng(SEED + requests)
    old = rng.integers(0, 30, requests).tolist()
    new = [int(rng.integers(0, 5)) if rng.random() < 0.95 else arc.PAGED_RELEASE for _ in old]
    new[0], new[-1] = 0, 4
    rows = sum(n for n in new if n != arc.PAGED_RELEASE) + 300
    assert rows > 4096
    p = PlanRun(old, new, 8, 5, rows, 4, 4000, seed=requests)
    same_plan(p.run(in_place), p.want())


@pytest.mark.parametrize("first", ["x", "q"])
@pytest.mark.parametrize("xt", [arc.F32, arc.F16])
def test_q_beside_the_rows_it_comes_from(xt, first):
    """x and q as columns of one wide row: q as in a buffer of its own, x and the columns between as they were."""
    kv, hpk, dim, N = 2, 3, 64, 9
    cols, width, size = (kv * hpk + 2 * kv) * dim, kv * hpk * dim, 4 if xt == arc.F32 else 2
    rng = np.random.default_rng(SEED)
    row = cols * size + width * 2 + 96  # bytes; 48 between the two, 48 behind
    x_at, q_at = (0, cols * size + 48) if first == "x" else (width * 2 + 48, 0)
    x = rng.standard_normal((N, cols)).astype(np.float32)
    xb = (x if xt == arc.F32 else pl.to_bits(x, xt)).view(np.uint8).reshape(N, -1)
    both = np.full((N, row), 0x5A, np.uint8)
    both[:, x_at: x_at + cols * size] = xb
    pool = [D(np.zeros((2, 16 * kv * dim), np.uint16)) for _ in range(2)]
    pages = arc.KvPages(pool[0], pool[1], 2, 16, kv, dim)
    batch = arc.PagedBatch(0, N, positions=D(np.arange(N, dtype=np.uint32) * 7), slots=D(np.arange(N, dtype=np.uint32) + 3))
    rope = arc.Rope(D(arc.rope_phases(dim, 1e4)[0]), dim)
    q = D(np.zeros((N, width), np.uint16))
    arc.rope_append(pages, batch, rope, xt, D(xb), cols, hpk, q, width)
    wide = D(both)
    arc.rope_append(pages, batch, rope, xt, wide.ptr + x_at, row // size, hpk, wide.ptr + q_at, row // 2)
    got = wide.download(np.uint8).reshape(N, row)
    both[:, q_at: q_at + width * 2] = q.download(np.uint8).reshape(N, -1)
    assert np.array_equal(got, both) and q.download(np.uint16).any()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("first", ["q", "out"])
def test_output_beside_q(first, new):
    """q and out as columns of one wide row."""
    s = pl.Step([100, 5], [new, 2], 16, 2, 2, 64, arc.F16, SEED + 1).upload()
    want = s.attention()[:, : s.width]
    ld = 2 * s.width + 16  # 8 columns between the two, 8 behind
    q_at, out_at = (0, s.width + 8) if first == "q" else (s.width + 8, 0)
    both = np.full((s.rows, ld), 0xABCD, np.uint16)
    both[:, q_at: q_at + s.width] = s.q[:, : s.width]
    wide = D(both)
    ws = arc.DeviceBuffer(arc.paged_attention_workspace_bytes(s.pages, s.batch, s.hpk))
    arc.paged_attention(s.pages, s.batch, wide.ptr + 2 * q_at, ld, s.hpk, wide.ptr + 2 * out_at, ld, ws)
    both[:, out_at: out_at + s.width] = want
    assert np.array_equal(wide.download(np.uint16).reshape(s.rows, ld), both)
