"""The paged-cache entry points on the GPU against float64 (paged_lib): the step's
plan bit for bit, rotary positions with the cache write, attention over pages."""
import numpy as np
import pytest
import torch

import arcllm_amd as arc
import paged_lib as pl

pytestmark = pytest.mark.gpu

SEED = 0x9A6ED
D = arc.DeviceBuffer.from_array
U32 = np.uint32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


# --------------------------------------------------------------------- plan
class PlanRun:
    def __init__(self, old, new, page, max_pages, rows, max_new, spare, num_pages=None, count=None, seed=0):
        rng = np.random.default_rng(SEED + seed)
        self.old, self.new, self.page, self.max_pages, self.rows, self.max_new = old, new, page, max_pages, rows, max_new
        held = [pl.pages_of(o, page) for o in old]
        need = sum(held) + spare
        self.num_pages = need if num_pages is None else num_pages
        order = rng.permutation(max(need, 1)).astype(U32)
        self.tables = rng.integers(0, 2 ** 32, (max(1, len(old)), max_pages), dtype=U32)
        at = 0
        for b, n in enumerate(held):
            n = min(n, max_pages)
            self.tables[b, :n] = order[at: at + n]
            at += n
        self.stack = np.zeros(max(1, self.num_pages), U32)
        free = order[at:][: self.num_pages]
        self.stack[: len(free)] = free
        self.count = len(free) if count is None else count
        B = len(old)
        self.d = dict(old=D(np.array(old + [0], U32)), new=D(np.array(new + [0], U32)), tables=D(self.tables),
                      stack=D(self.stack), count=D(np.array([self.count], U32)), count_out=arc.DeviceBuffer(4),
                      lens=arc.DeviceBuffer(4 * max(1, B)), starts=arc.DeviceBuffer(4 * (B + 1)),
                      positions=arc.DeviceBuffer(4 * max(1, rows)), slots=arc.DeviceBuffer(4 * max(1, rows)),
                      status=arc.DeviceBuffer(16))

    def run(self, in_place=False):
        d = self.d
        lens = d["old"] if in_place else d["lens"]
        batch = arc.PagedBatch(len(self.old), self.rows, self.max_pages, self.max_new, d["tables"], lens, d["starts"],
                               d["positions"], d["slots"])
        count_out = d["count"] if in_place else d["count_out"]
        arc.paged_plan(batch, d["old"], d["new"], self.page, d["stack"], self.num_pages, d["count"], count_out,
                       d["status"])
        B = len(self.old)
        get = lambda b, n: b.download(U32, n)  # noqa: E731
        return dict(tables=get(d["tables"], self.tables.size).reshape(self.tables.shape), lens=get(lens, B),
                    starts=get(d["starts"], B + 1), positions=get(d["positions"], self.rows),
                    slots=get(d["slots"], self.rows), stack=get(d["stack"], self.stack.size), count=int(get(count_out, 1)[0]),
                    status=get(d["status"], 4))

    def want(self):
        return pl.plan(self.old, self.new, self.page, self.tables, self.max_pages, self.rows, self.max_new, self.stack,
                       self.count, self.num_pages)


def same_plan(got, want):
    assert got["status"].tolist() == want["status"].tolist()
    for name in ("lens", "starts", "positions", "slots", "tables", "stack"):
        assert np.array_equal(got[name], want[name]), name
    assert got["count"] == want["count"]


R = arc.PAGED_RELEASE


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", ["one", "none", "zero", "grow", "border", "page1", "ended", "mixed", "wide", "many", "huge rows"])
def test_plan(name, in_place):
    rng = np.random.default_rng(SEED)
    kw = dict(page=16, max_pages=40, max_new=600, spare=50)
    if name == "one":
        old, new, kw["rows"] = [0], [1], 1
    elif name == "none":
        old, new, kw["rows"] = [], [], 5
    elif name == "zero":
        old, new, kw["rows"] = [5, 0, 16], [0, 0, 0], 2
    elif name == "grow":
        old, new, kw["rows"] = [15, 16, 17, 31], [1, 1, 1, 2], 5
    elif name == "border":
        old, new, kw["rows"] = [0, 624, 600], [600, 16, 40], 656
    elif name == "page1":
        kw.update(page=1, max_pages=9)
        old, new, kw["rows"] = [3, 0, 8], [2, 9, 1], 20
    elif name == "ended":
        old, new, kw["rows"] = [33, 64, 0, 10], [R, R, R, 40], 64
    elif name == "mixed":
        old = rng.integers(0, 300, 700).tolist()
        new = [int(rng.choice([0, 1, 1, 1, 7, 65])) if rng.random() < 0.9 else R for _ in old]
        kw.update(rows=sum(n for n in new if n != R) + 9, spare=4000)
    elif name == "wide":  # a long request among short ones, page ids far apart
        kw.update(page=4, max_pages=5000, max_new=9000, spare=3000)
        old, new = [1, 10000, 2, 0], [3, 9000, R, 1]
        kw["rows"] = 9100
    elif name == "many":  # several blocks of requests
        old = rng.integers(0, 40, 2500).tolist()
        new = [int(rng.integers(0, 4)) if rng.random() < 0.95 else R for _ in old]
        kw.update(page=8, rows=sum(n for n in new if n != R) + 700, spare=2600)
    else:
        old, new = [0, 100, 7], [20000, 1, 0]
        kw.update(max_pages=1300, max_new=20000, spare=1300, rows=70001)
    p = PlanRun(old, new, **kw)
    same_plan(p.run(in_place), p.want())
    if not in_place:  # the inputs are as they were: the same step again
        same_plan(p.run(), p.want())


@pytest.mark.parametrize("rows", [200, 5000])
@pytest.mark.parametrize("name,change,code", [
    ("no pages", dict(spare=3), arc.PLAN_NO_PAGES), ("table", dict(max_pages=2), arc.PLAN_TABLE),
    ("rows", dict(rows=20), arc.PLAN_TOKENS), ("max_new", dict(max_new=39), arc.PLAN_MAX_NEW),
    ("free list", dict(num_pages=9), arc.PLAN_FREE_LIST), ("free count", dict(count=1000), arc.PLAN_FREE_LIST),
    ("both", dict(max_pages=2, max_new=39), arc.PLAN_TABLE | arc.PLAN_MAX_NEW)])
def test_plan_refuses_a_step_whole(name, change, code, rows):
    kw = dict(page=8, max_pages=9, rows=rows, max_new=40, spare=9)
    kw.update(change)
    old, new = [9, 20, 8, 3], [40, 1, R, 0]
    if name == "free list":  # 9 pages of the pool, 9 free: the ended request's page has no place
        kw["spare"] = 9
    p = PlanRun(old, new, **kw)
    got = p.run()
    same_plan(got, p.want())
    assert got["status"][0] == code and got["lens"].tolist() == old
    assert not got["starts"].any() and np.all(got["slots"] == arc.NO_SLOT)


def test_plan_refuses_positions_past_31_bits():
    """Lengths whose sum with the new tokens passes 2^31 - 1 or 2^32 are not followed anywhere."""
    for old, new, max_pages in ((2 ** 31 - 1, 1, 2 ** 15), (2 ** 32 - 1, 5, 2 ** 15), (2 ** 32 - 40, R, 2 ** 15)):
        p = PlanRun([0], [1], 65536, 4, 8, 2 ** 32 - 2, 2)
        p.d["old"].upload(np.array([old, 0], U32))
        p.d["new"].upload(np.array([new, 0], U32))
        p.d["tables"].upload(p.tables)
        got = p.run()
        assert got["status"].tolist() == [arc.PLAN_TABLE, 0, 0, 0] and got["lens"].tolist() == [old]
        assert np.all(got["slots"] == arc.NO_SLOT) and np.array_equal(got["tables"], p.tables)


# --------------------------------------------------------------------- rope
def append_case(N, kv_heads, hpk, dim, rot, layout, xt, dtype, bias, page=16, ldx_pad=0, ldq_pad=0, stride_pad=0, far=5000, seed=0,
                **scaling):
    rng = np.random.default_rng(SEED + seed)
    heads = kv_heads * hpk
    cols = (heads + 2 * kv_heads) * dim
    ldx, ldq = cols + ldx_pad, heads * dim + ldq_pad
    x = (rng.standard_normal((N, ldx)) * 2).astype(np.float32)
    if xt == arc.F32:
        xv, xb = x[:, :cols].astype(np.float64), x
    else:
        xb = pl.to_bits(x, xt)
        xv = pl.from_bits(xb[:, :cols], xt)
    num_pages = pl.pages_of(N, page) + 2
    slots = rng.permutation(num_pages * page)[:N].astype(U32)
    if N > 4:
        slots[[1, N - 1]] = arc.NO_SLOT, num_pages * page  # padding, and the first number past the pool
    positions = rng.integers(0, far, N).astype(U32)
    positions[0] = 0
    b = [rng.standard_normal(n * dim).astype(np.float32) if bias else None for n in (heads, kv_heads, kv_heads)]
    phases, scale = arc.rope_phases(rot, 1e6, **scaling)
    stride = page * kv_heads * dim + stride_pad
    pool = [np.full((num_pages, stride), 0x1234, np.uint16) for _ in range(2)]
    dk, dv, dq = D(pool[0]), D(pool[1]), D(np.full((N, ldq), 0xABCD, np.uint16))
    pages = arc.KvPages(dk, dv, num_pages, page, kv_heads, dim, dtype, stride)
    batch = arc.PagedBatch(0, N, positions=D(positions), slots=D(slots))
    rope = arc.Rope(D(phases), rot, layout, scale)
    bd = [None if t is None else D(t) for t in b]
    arc.rope_append(pages, batch, rope, xt, D(xb), ldx, hpk, dq, ldq, q_bias=bd[0], k_bias=bd[1], v_bias=bd[2])
    q = dq.download(np.uint16).reshape(N, ldq)
    k, v = (t.download(np.uint16).reshape(num_pages, stride) for t in (dk, dv))
    # float64
    size = np.abs(xv)  # of the sum: bias + x round once in fp32
    if bias:
        full = np.concatenate(b).astype(np.float64)
        size = size + np.abs(full)
        xv = xv + full
    freqs, fscale = pl.rope_freqs(rot, 1e6, **scaling)
    h3, s3 = xv.reshape(N, -1, dim), size.reshape(N, -1, dim)
    turned, mag = pl.rotate(h3[:, : heads + kv_heads], positions, freqs, fscale, layout)
    # the pair's sizes for the additions' rounding
    _, mag_in = pl.rotate(s3[:, : heads + kv_heads], np.zeros(N, U32), freqs, fscale, layout)
    ref = np.concatenate([turned, h3[:, heads + kv_heads:]], 1)
    # errors before the rounding to 16 bits, relative to the pair's |a| + |b|: the addition 2^-24; the angle
    # 2 pi 2^-26; sincospi 4 ulp = 2^-22 of a value up to 1; scale and both products 2^-24 each
    fp32 = np.zeros_like(ref)
    fp32[:, : heads + kv_heads] = mag * (2 * np.pi * 2 ** -26 + 2 ** -22 + 4 * 2 ** -24) + mag_in * 2.0 ** -24
    fp32 += s3 * 2.0 ** -24
    u = pl.HALF_STEP[dtype]
    tol = u * (np.abs(ref) + fp32) + fp32 + (2.0 ** -25 if dtype == arc.F16 else 0)
    used = slots < num_pages * page
    err = lambda got, want, bound: float((np.abs(got - want) / bound).max()) if want.size else 0.0  # noqa: E731
    got_q = pl.from_bits(q[used, : heads * dim], dtype).reshape(-1, heads, dim)
    worst = err(got_q, ref[used, :heads], tol[used, :heads])
    assert np.all(q[~used] == 0xABCD) and np.all(q[:, heads * dim:] == 0xABCD)
    untouched = np.ones_like(k, bool)
    for t, at in ((k, heads), (v, heads + kv_heads)):
        for n in np.nonzero(used)[0]:
            pg, place = slots[n] // page, (slots[n] % page) * kv_heads * dim
            got = pl.from_bits(t[pg, place: place + kv_heads * dim], dtype).reshape(kv_heads, dim)
            worst = max(worst, err(got, ref[n, at: at + kv_heads], tol[n, at: at + kv_heads]))
            untouched[pg, place: place + kv_heads * dim] = False
        assert np.all(t[untouched] == 0x1234)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
@pytest.mark.parametrize("xt", [arc.F32, arc.F16, arc.BF16])
@pytest.mark.parametrize("layout", [arc.ROPE_INTERLEAVED, arc.ROPE_HALF])
def test_rope_types(layout, xt, dtype):
    append_case(37, 2, 3, 128, 128, layout, xt, dtype, bias=True, seed=1)


@pytest.mark.parametrize("layout", [arc.ROPE_INTERLEAVED, arc.ROPE_HALF])
@pytest.mark.parametrize("dim,rot", [(128, 8), (128, 24), (128, 64), (128, 120), (64, 64), (64, 8), (64, 40)])
def test_rope_part_of_the_head(dim, rot, layout):
    append_case(9, 1, 5, dim, rot, layout, arc.F32, arc.F16, bias=False, seed=2)


@pytest.mark.parametrize("kw", [dict(scaling=arc.ROPE_LINEAR, factor=8.0),
                                dict(scaling=arc.ROPE_YARN, factor=16.0, original_ctx=8192),
                                dict(freq_factors=np.linspace(1, 8, 64, dtype=np.float32))], ids=["linear", "yarn", "factors"])
@pytest.mark.parametrize("far", [300, 2 ** 20, 2 ** 31])
def test_rope_scaled_and_far(kw, far):
    append_case(21, 2, 2, 128, 128, arc.ROPE_HALF, arc.F32, arc.BF16, bias=True, far=far, seed=3, **kw)


@pytest.mark.parametrize("N,kv_heads,hpk,page", [(1, 1, 1, 1), (2, 4, 7, 16), (3, 256, 1, 8), (5, 1, 64, 65536), (600, 3, 2, 32)])
def test_rope_sizes_and_strides(N, kv_heads, hpk, page):
    append_case(N, kv_heads, hpk, 64, 64, arc.ROPE_INTERLEAVED, arc.F32, arc.F16, bias=True, page=page, ldx_pad=24, ldq_pad=40,
                stride_pad=72, seed=4)


def test_rope_more_rows_than_a_grid_holds():
    """70001 rows of one small head each: the rows past the grid's second dimension."""
    append_case(70001, 1, 1, 64, 16, arc.ROPE_HALF, arc.F16, arc.F16, bias=False, page=64, seed=5)


# ---------------------------------------------------------------- attention
TYPES = [arc.F16, arc.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,hpk", [(1, 1), (4, 7), (2, 8), (3, 5), (1, 33), (1, 64)])
def test_heads(kv_heads, hpk, dim, dtype):
    s = pl.Step([200, 0, 37, 63], [1, 3, 40, 1], 16, kv_heads, hpk, dim, dtype, SEED + 1).upload()
    s.check(s.attention())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 511, 513, 1000, 2047, 4099])
def test_decode_lengths(T, dtype):
    s = pl.Step([T - 1], [1], 16, 2, 4, 128, dtype, SEED + T).upload()
    s.check(s.attention())


@pytest.mark.parametrize("M", [2, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("old", [0, 1, 77])
def test_chunk_lengths(M, old):
    s = pl.Step([old], [M], 16, 1, 4, 128, arc.F16, SEED + M + old).upload()
    s.check(s.attention())


@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 128, 1024, 65536])
def test_page_sizes(page):
    s = pl.Step([300, 11], [1, 70], page, 1, 4, 64, arc.F16, SEED + page, spare=0 if page > 1024 else 2).upload()
    s.check(s.attention())


def test_ragged_batch_rows_behind_and_strides():
    """Requests of no new tokens and of no positions among the others, rows behind the last, gaps between
    rows and pages."""
    old = [0, 500, 3, 0, 129, 1, 64, 0]
    new = [5, 1, 0, 0, 40, 1, 64, 1]
    s = pl.Step(old, new, 16, 2, 3, 128, arc.BF16, SEED + 5, rows=sum(new) + 13, stride_pad=40, ld_pad=24).upload()
    s.check(s.attention())


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 2), (64, 0), (64, 4), (100, 64), (100, 65), (1000, 4), (128, 700),
                                          (2 ** 32 - 1, 2 ** 32 - 1), (5, 2 ** 32 - 1), (0, 9)])
@pytest.mark.parametrize("dim", [64, 128])
def test_window_and_sinks(window, sinks, dim):
    s = pl.Step([900, 0, 130, 20], [1, 90, 150, 3], 16, 2, 4, dim, arc.F16, SEED + 6).upload()
    s.check(s.attention(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(512, 4), (4096, 130)])
def test_window_far_behind(window, sinks):
    """Only the window's and the sinks' pages are read: every other table entry is no page of the pool."""
    s = pl.Step([20000, 9000], [1, 30], 16, 1, 4, 128, arc.F16, SEED + 7)
    for b in range(2):
        first = max(0, s.old[b] + 1 - window) // 16
        s.tables[b, -(-sinks // 16): first] = 0xFFFFFFFF
    s.upload()
    s.check(s.attention(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scale(scale):
    s = pl.Step([100], [20], 16, 2, 2, 64, arc.F16, SEED + 8).upload()
    s.check(s.attention(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_sharp_key_and_thousands_of_faint_ones(dtype):
    """Weights far below the largest, under fp16's normal range: they count."""
    s = pl.Step([3999], [1], 16, 1, 2, 128, dtype, SEED + 9)
    s.q[:] = pl.to_bits(np.ones(s.q.shape), dtype)
    faint = pl.to_bits(np.full(s.kvd, -0.6), dtype)  # scores -0.6 sqrt(128) = -6.8 against 4.5
    sharp = pl.to_bits(np.full(s.kvd, 0.4), dtype)
    for p in range(4000):
        row = sharp if p == 1234 else faint
        s.k[s.tables[0, p // 16], (p % 16) * s.kvd: (p % 16 + 1) * s.kvd] = row
        s.K[0][p] = pl.from_bits(row, dtype).reshape(1, 128)
    s.upload()
    s.check(s.attention())


def test_scores_that_grow_and_fall_along_the_context():
    """The running maximum moves in every block, or never after the first."""
    for sign in (1.0, -1.0):
        s = pl.Step([1500, 700], [1, 60], 16, 1, 3, 128, arc.F16, SEED + 10)
        s.q[:] = pl.to_bits(np.ones(s.q.shape), arc.F16)
        for b, n in enumerate((1501, 760)):
            for p in range(n):
                row = pl.to_bits(np.full(s.kvd, sign * (p / n - 0.5) * 4), arc.F16)
                s.k[s.tables[b, p // 16], (p % 16) * s.kvd: (p % 16 + 1) * s.kvd] = row
                s.K[b][p] = pl.from_bits(row, arc.F16).reshape(1, 128)
        s.upload()
        s.check(s.attention())


def test_pages_outside_the_pool_are_not_read():
    """Table entries that name no page: their positions are not seen; a row that sees none is zero."""
    s = pl.Step([200, 40, 64], [1, 20, 1], 16, 2, 2, 128, arc.F16, SEED + 11)
    dropped = [np.zeros(n, bool) for n in s.lens]
    for b, entry, value in ((0, 3, s.num_pages), (0, 12, 0xFFFFFFFF), (1, 0, s.num_pages + 5), (2, 0, 2 ** 31)):
        s.tables[b, entry] = value
        dropped[b][entry * 16: entry * 16 + 16] = True
    for entry in range(1, 5):
        s.tables[2, entry] = 0xFFFFFFF0
        dropped[2][entry * 16: entry * 16 + 16] = True
    s.upload()
    bits = s.attention()
    s.check(bits, dropped=dropped)
    assert not bits[int(s.starts[2]), : s.width].any()


def test_lens_beyond_the_table_and_starts_beyond_the_rows():
    """A length past the table's row is cut there, one short of the new tokens leaves rows without a
    position (zeros): nothing outside the arrays is read or written."""
    s = pl.Step([30, 5], [2, 3], 16, 1, 2, 64, arc.F16, SEED + 12, max_pages=2)
    s.lens[:] = 1000, 2  # the table holds 32 = 30 + 2; the second request's first row lies at position -1
    s.upload()
    bits = s.attention()
    good = pl.Step([30, 5], [2, 3], 16, 1, 2, 64, arc.F16, SEED + 12, max_pages=2)
    good.check(bits, rows={0, 1})
    assert not bits[2, : s.width].any() and np.all(np.isfinite(pl.from_bits(bits[3:5, : s.width], arc.F16)))
    s.dstarts.upload(np.array([0, 2, 900], U32))  # 898 new tokens, 5 rows
    bits = s.attention()
    assert np.all(bits[:, s.width:] == 0xABCD)
    good.check(bits, rows={0, 1})


def test_infinities_and_nan_where_nothing_is_seen():
    """Positions behind a token, outside its window, in unused places of its pages and of the others."""
    s = pl.Step([70], [30], 16, 1, 4, 128, arc.F16, SEED + 13)
    # the last 20 new tokens and the first 9 positions: rows 0..9 with a window of 40 see neither
    for p in list(range(9)) + list(range(80, 100)):
        for t, bad in ((s.k, 0x7C00), (s.v, 0xFC00)):
            t[s.tables[0, p // 16], (p % 16) * s.kvd: (p % 16 + 1) * s.kvd] = bad if p % 2 else 0x7E00
    s.upload()
    bits = s.attention(window=40)
    s.check(bits, window=40, rows=set(range(10)))


def test_long_context_offsets_pass_32_bits():
    """A pool whose pages lie 2^29 elements apart: offsets of 2^32 elements and more."""
    page, kv, dim, n = 16, 1, 128, 180
    s = pl.Step([n - 4], [4], page, kv, 2, dim, arc.F16, SEED + 14, spare=0)
    s.upload()
    stride = 1 << 29
    k = torch.zeros(s.num_pages * stride, dtype=torch.int16, device="cuda")
    v = torch.zeros(s.num_pages * stride, dtype=torch.int16, device="cuda")
    for t, src in ((k, s.k), (v, s.v)):
        t.view(s.num_pages, stride)[:, : page * kv * dim] = torch.from_numpy(src.view(np.int16)).cuda()
    torch.cuda.synchronize()
    s.pages = arc.KvPages(k.data_ptr(), v.data_ptr(), s.num_pages, page, kv, dim, arc.F16, stride)
    s.check(s.attention())


@pytest.mark.parametrize("dtype", TYPES)
def test_many_requests(dtype):
    rng = np.random.default_rng(SEED)
    old = rng.integers(0, 400, 150).tolist()
    new = [1 if rng.random() < 0.9 else int(rng.integers(0, 40)) for _ in old]
    s = pl.Step(old, new, 16, 2, 4, 64, dtype, SEED + 15).upload()
    s.check(s.attention())


def test_same_call_twice_gives_the_same_bits():
    s = pl.Step([5000, 100, 0], [1, 30, 200], 16, 4, 7, 128, arc.BF16, SEED + 16).upload()
    ws = arc.DeviceBuffer(arc.paged_attention_workspace_bytes(s.pages, s.batch, s.hpk))
    a = s.attention(workspace=ws)
    assert np.array_equal(a, s.attention(workspace=ws))


def test_long_chunk_rows_sampled():
    s = pl.Step([1000, 3000], [700, 1], 16, 2, 7, 128, arc.F16, SEED + 17).upload()
    s.check(s.attention(), rows={0, 1, 17, 18, 19, 255, 256, 350, 511, 640, 698, 699, 700})


def test_long_decode_is_split():
    s = pl.Step([40000, 12345], [1, 1], 64, 1, 8, 128, arc.F16, SEED + 18).upload()
    s.check(s.attention())


def test_session_cache_as_pages():
    """A contiguous cache is a pool whose pages lie in order: the same rows as arc_prefill_attention's
    (fp16 outputs of the same sums, each within the bound of its own)."""
    T, M, kv, hpk = 333, 45, 2, 4
    s = pl.Step([T - M], [M], 16, kv, hpk, 128, arc.F16, SEED + 19)
    n = s.num_pages
    flat = [np.zeros((n * 16, s.kvd), np.uint16) for _ in range(2)]
    for f, t in zip(flat, (s.k, s.v)):
        for p in range(T):
            f[p] = t[s.tables[0, p // 16], (p % 16) * s.kvd: (p % 16 + 1) * s.kvd]
    s.k, s.v = (f.reshape(n, 16 * s.kvd) for f in flat)
    s.tables[0] = np.arange(s.max_pages)
    s.upload()
    bits = s.attention()
    s.check(bits)
    x = arc.DeviceBuffer(M * s.width * 2)
    arc.prefill_attention(D(pl.from_bits(s.q, arc.F16).astype(np.float32)), s.dk, s.dv, kv, hpk, T, T - M, M, x, s.width)
    other = x.download(np.uint16).reshape(M, s.width)
    s.check(other)


# ------------------------------------------------------------------ together
def test_a_layer_as_a_server_runs_it():
    """Three steps of an attention layer for three requests: plan, q|k|v projection, bias + rope + cache
    write, attention, o projection.  Each step's attention is held to float64 of what the rope step left, and
    the cache to float64 of the projections."""
    H, kv, hpk, dim, page = 512, 2, 2, 128, 16
    kvd, cols = kv * dim, 512 + 2 * 256
    rng = np.random.default_rng(SEED)
    wq, wk, wv, wo = (arc.synth_packed(arc.Q4_K, SEED, i, n, H) for i, n in enumerate((H, kvd, kvd, H)))
    dw = [D(w) for w in (wq, wk, wv, wo)]
    bias = [rng.standard_normal(n).astype(np.float32) for n in (H, kvd, kvd)]
    db = [D(b) for b in bias]
    num_pages, max_pages, rows = 24, 8, 80
    dk, dv = (D(np.full((num_pages, page * kvd), 0x7E00, np.uint16)) for _ in range(2))
    pages = arc.KvPages(dk, dv, num_pages, page, kv, dim, arc.F16)
    phases, scale = arc.rope_phases(dim, 1e6)
    dphases = D(phases)
    rope = arc.Rope(dphases, dim, arc.ROPE_INTERLEAVED, scale)
    tables, lens, starts = (arc.DeviceBuffer(4 * n) for n in (3 * max_pages, 3, 4))
    lens.zero()
    positions, slots = arc.DeviceBuffer(4 * rows), arc.DeviceBuffer(4 * rows)
    stack, count, status = D(np.arange(num_pages, dtype=U32)), D(np.array([num_pages], U32)), arc.DeviceBuffer(16)
    batch = arc.PagedBatch(3, rows, max_pages, 64, tables, lens, starts, positions, slots)
    ws = arc.DeviceBuffer(arc.paged_attention_workspace_bytes(pages, batch, hpk))
    gw = arc.DeviceBuffer(max(arc.prefill_gemm_workspace_bytes(cols, H), arc.prefill_gemm_workspace_bytes(H, H)))
    y, q, o, z = (arc.DeviceBuffer(rows * n) for n in (cols * 4, H * 2, H * 2, H * 4))
    freqs, _ = pl.rope_freqs(dim, 1e6)
    wo64 = np.empty((H, H), np.float32)
    dd = arc.DeviceBuffer(H * H * 4)
    arc.dequant(arc.Q4_K, dw[3], H, H, dd)
    wo64 = dd.download(np.float32).reshape(H, H).astype(np.float16).astype(np.float64)
    held = [0, 0, 0]
    K, V = [np.zeros((0, kv, dim)) for _ in held], [np.zeros((0, kv, dim)) for _ in held]
    for new in ([33, 1, 0], [1, 5, 40], [1, arc.PAGED_RELEASE, 1]):
        fresh = [0 if n == arc.PAGED_RELEASE else n for n in new]
        x = rng.standard_normal((rows, H)).astype(np.float16)
        arc.paged_plan(batch, lens, D(np.array(new, U32)), page, stack, num_pages, count, count, status)
        arc.prefill_qkv(dw[0], dw[1], dw[2], arc.Q4_K, H, kvd, H, D(x), rows, y, gw)
        arc.rope_append(pages, batch, rope, arc.F32, y, cols, hpk, q, H, *db)
        arc.paged_attention(pages, batch, q, H, hpk, o, H, ws)
        arc.prefill_gemm(arc.Q4_K, dw[3], H, H, o, rows, z, gw)
        used = sum(fresh)
        assert status.download(U32).tolist()[:3] == [0, 0, used]
        y_h = y.download(np.float32).reshape(rows, cols).astype(np.float64)
        q_h = pl.from_bits(q.download(np.uint16), arc.F16).reshape(rows, 4, dim)
        o_h = pl.from_bits(o.download(np.uint16), arc.F16).reshape(rows, 4, dim)
        z_h = z.download(np.float32).reshape(rows, H)
        sl = slots.download(U32)
        kc, vc = (pl.from_bits(t.download(np.uint16), arc.F16).reshape(-1, kv, dim) for t in (dk, dv))
        n = 0
        for b in range(3):
            if new[b] == arc.PAGED_RELEASE:
                held[b], K[b], V[b] = 0, K[b][:0], V[b][:0]
                continue
            r = slice(n, n + fresh[b])
            pos = np.arange(held[b], held[b] + fresh[b]).astype(U32)
            full = (y_h[r] + np.concatenate(bias)).reshape(-1, 8, dim)
            turned, _ = pl.rotate(full[:, :6], pos, freqs, 1.0, arc.ROPE_INTERLEAVED)
            assert np.abs(q_h[r] - turned[:, :4]).max(initial=0) <= 2.0 ** -11 * 1.01 * max(1.0, np.abs(turned).max(initial=0))
            at = sl[r].astype(int)
            assert np.abs(kc[at] - turned[:, 4:]).max(initial=0) <= 2.0 ** -11 * 1.01 * max(1.0, np.abs(turned).max(initial=0))
            K[b], V[b] = np.concatenate([K[b], kc[at]]), np.concatenate([V[b], vc[at]])
            held[b] += fresh[b]
            vmax = np.abs(V[b]).max(initial=0)
            for i in range(fresh[b]):
                ref, mass, off, seen = pl.attend(q_h[n + i], K[b], V[b], int(pos[i]), dim ** -0.5)
                assert np.all(np.abs(o_h[n + i] - ref) <= pl.attention_bound(ref, mass, off, seen, vmax, arc.F16)), (b, i)
            n += fresh[b]
        want = o_h[:used].reshape(used, H) @ wo64.T
        assert np.abs(z_h[:used] - want).max() <= 1e-3 * np.abs(want).max()
        # the tables hold exactly the pages of the positions, no page twice
        t = tables.download(U32).reshape(3, max_pages)
        own = [p for b in range(3) for p in t[b, : pl.pages_of(held[b], page)].tolist()]
        left = count.download(U32)[0]
        own += stack.download(U32)[:left].tolist()
        assert sorted(own) == list(range(num_pages))


class TorchStream:
    """torch's current stream as the framework's."""

    @property
    def handle(self):
        return torch.cuda.current_stream().cuda_stream


def test_captured_step_replays():
    """A decode step captured once (plan in place, rope, attention) and replayed: each replay advances the
    lengths by itself and equals the eager step of a second state, with eager work and synchronizations
    between the replays."""
    kv, hpk, dim, page, B = 2, 4, 64, 4, 3
    rng = np.random.default_rng(SEED + 21)
    cols, width = (kv * hpk + 2 * kv) * dim, kv * hpk * dim
    num_pages, max_pages = 40, 12
    x0 = rng.standard_normal((6, B, cols)).astype(np.float32)

    def state():
        s = dict(k=torch.zeros(num_pages, page * kv * dim, dtype=torch.float16, device="cuda"),
                 tables=torch.zeros(B, max_pages, dtype=torch.int32, device="cuda"),
                 lens=torch.zeros(B, dtype=torch.int32, device="cuda"), starts=torch.zeros(B + 1, dtype=torch.int32, device="cuda"),
                 positions=torch.zeros(B, dtype=torch.int32, device="cuda"), slots=torch.zeros(B, dtype=torch.int32, device="cuda"),
                 new=torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda"),
                 stack=torch.arange(num_pages, dtype=torch.int32, device="cuda"),
                 count=torch.tensor([num_pages], dtype=torch.int32, device="cuda"),
                 status=torch.zeros(4, dtype=torch.int32, device="cuda"),
                 x=torch.zeros(B, cols, device="cuda"), q=torch.zeros(B, width, dtype=torch.float16, device="cuda"),
                 out=torch.zeros(B, width, dtype=torch.float16, device="cuda"),
                 phases=torch.from_numpy(arc.rope_phases(dim, 1e4)[0].view(np.int64)).cuda())
        s["v"] = torch.zeros_like(s["k"])
        p = lambda n: s[n].data_ptr()  # noqa: E731
        s["pages"] = arc.KvPages(p("k"), p("v"), num_pages, page, kv, dim)
        s["batch"] = arc.PagedBatch(B, B, max_pages, 1, p("tables"), p("lens"), p("starts"), p("positions"), p("slots"))
        s["ws"] = torch.full((arc.paged_attention_workspace_bytes(s["pages"], s["batch"], hpk),), 255, dtype=torch.uint8,
                             device="cuda")
        return s

    def step(s):
        st, p = TorchStream(), lambda n: s[n].data_ptr()  # noqa: E731
        arc.paged_plan(s["batch"], p("lens"), p("new"), page, p("stack"), num_pages, p("count"), p("count"), p("status"),
                       stream=st)
        arc.rope_append(s["pages"], s["batch"], arc.Rope(p("phases"), dim), arc.F32, p("x"), cols, hpk, p("q"), width, stream=st)
        arc.paged_attention(s["pages"], s["batch"], p("q"), width, hpk, p("out"), width, p("ws"), stream=st)

    a, b = state(), state()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step(a)
    torch.cuda.synchronize()
    for i in range(6):
        for s in (a, b):
            s["x"].copy_(torch.from_numpy(x0[i]))
        step(b)
        g.replay()
        torch.cuda.synchronize()
        assert a["status"].tolist()[0] == 0 and a["lens"].tolist() == [i + 1] * B
        for name in ("tables", "lens", "starts", "slots", "count", "q", "k", "v", "out"):
            assert torch.equal(a[name], b[name]), (i, name)
        assert float(a["out"].float().abs().max()) > 0


def test_calls_on_their_own_streams():
    """Two steps at once, each on a stream and workspace of its own."""
    a = pl.Step([3000, 20], [1, 50], 16, 2, 4, 128, arc.F16, SEED + 22).upload()
    b = pl.Step([700], [130], 32, 1, 7, 64, arc.BF16, SEED + 23).upload()
    arc.synchronize()
    sa, sb = arc.Stream(), arc.Stream()
    outs = []
    for s, st in ((a, sa), (b, sb)) * 3:
        ws = arc.DeviceBuffer(arc.paged_attention_workspace_bytes(s.pages, s.batch, s.hpk))
        out = D(np.full((s.rows, s.ldo), 0xABCD, np.uint16))
        arc.synchronize()
        outs.append((s, st, ws, out))
    for s, st, ws, out in outs:
        arc.paged_attention(s.pages, s.batch, s.dq, s.ldq, s.hpk, out, s.ldo, ws, stream=st)
    sa.synchronize()
    sb.synchronize()
    for s, _, _, out in outs:
        s.check(out.download(np.uint16).reshape(s.rows, s.ldo))
