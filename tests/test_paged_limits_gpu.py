"""Paged attention at its edges: infinities and NaN that some rows see and others do not,
the last position, many requests, a wrong max_new, negative scales, the workspace's size."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_lib as pl

pytestmark = pytest.mark.gpu

SEED = 0x11A17
D = arc.DeviceBuffer.from_array
INF = {arc.F16: 0x7C00, arc.BF16: 0x7F80}
NAN = {arc.F16: 0x7E01, arc.BF16: 0x7FC1}


def put(s, b, t, pos, head, dim, bits):
    t[s.tables[b, pos // s.page], (pos % s.page) * s.kvd + head * s.dim + dim] = bits


def rows_of(s, bits):
    return pl.from_bits(bits[: s.used, : s.width], s.dtype).reshape(s.used, s.heads, s.dim)


@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dim, new, dtype):
    """+inf, -inf and NaN of V at single dims of one kv head: exactly the rows whose token is at or behind the
    position, in that kv head's query heads, have them there (weights are positive); every other value is
    as without them.  Old positions (all rows see them) and new ones (the later rows do)."""
    old = 70
    s = pl.Step([old, 40], [new, new], 16, 2, 4, dim, dtype, SEED + new)
    clean = pl.Step([old, 40], [new, new], 16, 2, 4, dim, dtype, SEED + new).upload()
    want = rows_of(s, clean.attention())
    marks = [(3, 0, 5, INF[dtype], np.inf), (old + new // 2, 1, dim - 1, INF[dtype] | 0x8000, -np.inf),
             (old + new - 1, 0, 17, NAN[dtype], np.nan), (old // 2, 1, 0, NAN[dtype], np.nan)]
    for pos, head, d, bits, _ in marks:
        put(s, 0, s.v, pos, head, d, bits)
    got = rows_of(s, s.upload().attention())
    for pos, head, d, _, value in marks:
        for i in range(new):
            if old + i >= pos:
                want[i, head * 4: head * 4 + 4, d] = value
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("new", [1, 40])
def test_not_finite_beside_a_page_that_is_none(new):
    """The same in a unit of which some positions have no page."""
    s = pl.Step([100], [new], 16, 1, 4, 64, arc.F16, SEED)
    s.tables[0, 2] = 0xFFFFFFFF
    bits = s.upload().attention()
    dropped = [np.zeros(100 + new, bool)]
    dropped[0][32:48] = True
    s.check(bits, dropped=dropped)
    want = rows_of(s, bits)
    put(s, 0, s.v, 20, 0, 9, INF[arc.F16])
    want[:, :, 9] = np.inf
    assert np.array_equal(rows_of(s, s.upload().attention()), want)


def test_nan_in_k_reaches_the_rows_that_see_it():
    s = pl.Step([50], [30], 16, 2, 2, 64, arc.F16, SEED + 1)
    put(s, 0, s.k, 65, 1, 3, NAN[arc.F16])  # new token 15, kv head 1
    got = rows_of(s, s.upload().attention())
    assert np.isnan(got[15:, 2:]).all() and np.isfinite(got[:15]).all() and np.isfinite(got[:, :2]).all()


def test_the_last_position():
    """A request of 2^31 - 1 positions, the most there are, with a window: only its last page is read, the
    pool holds no other.  One of 2^31 is taken as that."""
    page, dim, window = 65536, 64, 100
    s = pl.Step([page - 2], [1], page, 1, 2, dim, arc.F16, SEED + 2, spare=0)  # the last page's positions
    s.k[:], s.v[:] = np.nan_to_num(pl.from_bits(s.k, arc.F16)).astype(np.float16).view(np.uint16), \
        np.nan_to_num(pl.from_bits(s.v, arc.F16)).astype(np.float16).view(np.uint16)
    want = s.upload().attention(window=window)
    s.check(want, window=window)
    s.max_pages = 2 ** 31 // page
    s.tables = np.full((1, s.max_pages), 0xFFFFFFFF, np.uint32)
    s.tables[0, -1] = 0
    for held in (2 ** 31 - 1, 2 ** 31):
        s.lens = np.array([held], np.uint32)
        assert np.array_equal(s.upload().attention(window=window), want), held


@pytest.mark.parametrize("requests", [64, 65, 256, 257, 1100])
def test_requests_around_the_walks_blocks(requests):
    """Most without new tokens, so that parts of the work begin far into the batch."""
    rng = np.random.default_rng(SEED + requests)
    old = [int(rng.integers(0, 90)) for _ in range(requests)]
    new = [0] * requests
    for b in list(rng.choice(requests, 20, replace=False)) + [0, requests - 1]:
        new[b] = int(rng.choice([1, 1, 2, 45]))
    s = pl.Step(old, new, 16, 2, 4, 64, arc.F16, SEED + requests).upload()
    s.check(s.attention())


def test_no_request_has_new_tokens():
    s = pl.Step([10, 20], [0, 0], 16, 1, 2, 64, arc.F16, SEED + 3, rows=5).upload()
    s.check(s.attention())


@pytest.mark.parametrize("max_new", [0, 1, 7, 4096])
def test_max_new_decides_speed_only(max_new):
    """Too small or too large a bound: the same rows within the bound."""
    s = pl.Step([300, 5, 0], [1, 60, 33], 16, 2, 4, 128, arc.F16, SEED + 4, max_new=max_new).upload()
    s.check(s.attention())


@pytest.mark.parametrize("rows", [61, 70])
def test_rows_of_no_request_among_many(rows):
    """tokens that leave every request many rows if all are used: one request has only a few of them."""
    s = pl.Step([90, 200], [60, 1], 16, 1, 8, 64, arc.F16, SEED + 5, rows=rows).upload()
    s.check(s.attention())


@pytest.mark.parametrize("new", [1, 50])
def test_negative_scale(new):
    s = pl.Step([200], [new], 16, 1, 4, 64, arc.BF16, SEED + 6).upload()
    s.check(s.attention(scale=-0.2), scale=-0.2)


def test_workspace_grows_with_the_step_and_stays_bounded():
    p = arc.KvPages(1 << 20, 1 << 21, 4, 16, 8, 128)
    size = [arc.paged_attention_workspace_bytes(p, arc.PagedBatch(4, n), 4) for n in (0, 1, 8, 9, 64, 4096, 1 << 20)]
    assert size == sorted(size) and size[0] > 0 and size[-1] == size[-2] < 256 << 20


@pytest.mark.parametrize("hpk,new,dim", [(8, 1, 128), (5, 200, 128), (8, 77, 64)])
def test_nothing_is_written_behind_the_workspace(hpk, new, dim):
    """A workspace of exactly the stated size, at the end of a larger buffer's first part: the rest keeps
    its contents.  Contexts long enough that every part of the work is cut."""
    s = pl.Step([9000, 8000], [new, 1], 16, 2, hpk, dim, arc.F16, SEED + 7).upload()
    n = arc.paged_attention_workspace_bytes(s.pages, s.batch, hpk)
    ws = D(np.full(n + 4096, 0x5A, np.uint8))
    bits = s.attention(workspace=ws)
    s.check(bits, rows={0, new // 2, new - 1, new})
    assert np.all(ws.download(np.uint8)[n:] == 0x5A)


@pytest.mark.parametrize("kv_heads,dim,old,new", [(256, 64, [70, 0, 33], [1, 2, 40]), (97, 128, [40, 9], [1, 35]),
                                                  (255, 64, [0], [1])])
def test_many_kv_heads(kv_heads, dim, old, new):
    """Parts that begin and end at any of them."""
    s = pl.Step(old, new, 16, kv_heads, 1, dim, arc.F16, SEED + kv_heads).upload()
    s.check(s.attention())


@pytest.mark.parametrize("new,hpk,dim,window,max_new", [(1300, 64, 64, 0, None), (1300, 64, 64, 100, None),
                                                        (5000, 16, 128, 0, None), (5000, 16, 128, 700, None),
                                                        (200, 64, 64, 0, 0), (200, 64, 128, 9, 0)])
def test_more_tiles_than_a_wave_has_lanes(new, hpk, dim, window, max_new):
    """Of 128, 256 and 32 rows: each row is some tile's, wherever the parts are cut."""
    s = pl.Step([150, 3], [new, 2], 32, 2, hpk, dim, arc.BF16, SEED + new, max_new=max_new).upload()
    bits = s.attention(window=window)
    assert not np.any(np.all(bits[: s.used, : s.width].reshape(s.used, -1, dim) == 0xABCD, axis=2))
    s.check(bits, window=window, rows={0, 1, 2, 3, 63, 64, 65, 127, new // 2, new - 2, new - 1, new, new + 1})
