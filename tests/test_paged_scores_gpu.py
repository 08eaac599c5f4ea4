"""Paged attention where scores are large or weights faint: finite scores of any size in fp32."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_exact as px

pytestmark = pytest.mark.gpu

SEED = 0x5C0BE


def large_step(old, new, kv_heads, dim, dtype, exponent, order):
    """Scores of about 2^exponent powers of two, exact in fp32: q = (+-A, 2^8) and k = (B, i 2^n) in two dims, A B =
    1.4375 2^30 and i 2^(n+8), i = 0 .. 11, a multiple of 2^10 where fp32's step is 2^7.  The scale makes
    a step of i worth 1.44 powers of two, or 2^10 as many as the scale gives it.  Four heads: A, -A, 0, A.
    order: keys with k = (0, ..) among them, whose scores are small: none, the first, the last."""
    rng = np.random.default_rng(SEED + exponent)
    s = px.GivenStep(old, new, 16, kv_heads, 4, dim, dtype, SEED + exponent)
    q = np.zeros((4, dim))
    q[:, 0] = np.array([1.0, -1.0, 0.0, 1.0]) * 1.4375 * 2 ** 15
    q[:, dim // 2] = 2.0 ** 8
    s.give_q(np.tile(q, (kv_heads, 1)))
    unit = 2.0 ** max(10, 31 - exponent) if exponent < 21 else 2.0 ** 10
    for b, n in enumerate(s.lens):
        n = int(n)
        k = np.zeros((n, kv_heads, dim))
        small = {"none": 0, "first": n // 2, "last": n // 3}[order]
        k[:, :, 0] = 2.0 ** 15
        k[:small, :, 0] = 0.0
        k[:, :, dim // 2] = rng.integers(0, 12, (n, kv_heads)) * unit / 2 ** 8
        s.give(b, k[::-1] if order == "last" else k)
    return s.upload(), 2.0 ** (exponent - 31)


@pytest.mark.parametrize("order", ["none", "first", "last"])
@pytest.mark.parametrize("exponent", [11, 13, 20, 26, 29, 32, 100, 140])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
def test_large_scores(dtype, dim, exponent, order):
    """A few rows of short and cut contexts, many rows of one tile and of cut ones.  Sums of 3000 positions at most:
    with 16 values a step no more than 3100 additions."""
    for old, new, kv_heads in (([40, 2990], [1, 3], 1), ([30, 7], [12, 1], 1), ([2400], [50], 1), ([0, 20], [40, 33], 140)):
        s, scale = large_step(old, new, kv_heads, dim, dtype, exponent, order)
        last = sum(new) - 1
        s.check_exact(s.attention(scale=scale), scale, 3100, rows={0, 1, last // 2, last})


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("value", [1.0, 100.0, 8000.0])
@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
def test_one_key_is_the_answer(dtype, value, new):
    """q and k constant, the default scale: whatever the score, rows of equal scores are the mean of V, and the
    first, which sees one position, is its V."""
    s = px.GivenStep([0], [new], 16, 1, 2, 128, dtype, SEED)
    s.give_q(value)
    s.give(0, np.full((new, 1, 128), value))
    bits = s.upload().attention()
    s.check_exact(bits, 128 ** -0.5, 64)
    assert np.array_equal(bits[0].reshape(2, 128), s.v[s.tables[0, 0], :128][None].repeat(2, 0))


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_as_large_as_fp32_holds(new, sign):
    """bf16 scores of 128 2^60 2^60 = 2^127, all equal, of either sign."""
    s = px.GivenStep([300], [new], 16, 1, 2, 128, arc.BF16, SEED + 1)
    s.give_q(sign * 2.0 ** 60)
    s.give(0, np.full((300 + new, 1, 128), 2.0 ** 60))
    for scale in (2.0 ** -60, 1.0, 2.0 ** 60):
        s.check_exact(s.upload().attention(scale=scale), scale, 400)


@pytest.mark.parametrize("new,requests,dim", [(1, 1, 64), (1, 64, 64), (40, 1, 128), (40, 96, 64), (40, 32, 128)])
@pytest.mark.parametrize("below", [14.5, 18.7, 20.35, 23.6, 24.6, 25.01, 28.7])
@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
def test_one_sharp_key_before_a_long_context(dtype, below, new, requests, dim):
    """131071 positions, one of them `below` powers of two above all others, V = 1: rows are 1.  The faint keys all
    round alike, so theirs is one rounding 131070 times.  Many requests share the pages, one of faint keys over
    and over and one with the sharp one: a tile is one part then and its sums go over the whole context, one addition for
    16 positions at most."""
    n, page, kv = 131071, 64, 8
    s = px.GivenStep([2 * page - new] + [0] * (requests - 1), [new] * requests, page, kv, 1, dim, dtype, SEED + 2)
    s.give_q(1.0)
    k = np.zeros((2 * page, kv, dim))
    k[page + 9] = 1.0
    s.give(0, k, np.ones(k.shape))
    faint, sharp = s.tables[0, :2]
    s.max_pages, s.lens[:] = 2048, n
    s.tables = np.full((requests, 2048), faint, np.uint32)
    s.tables[:, 12] = sharp
    scale = float(np.float32(below / (dim * px.LOG2E)))
    bits = s.upload().attention(scale=scale)
    x = np.zeros((n, dim))
    x[12 * page + 9] = 1.0
    ref, tol = px.exact_row(np.ones((1, dim)), x, np.ones((n, dim)), scale, n // 16, dtype)
    assert np.abs(ref - 1).max() < 1e-9
    err = np.abs(px.pl.from_bits(bits, dtype) - 1.0).max()
    assert err <= tol.max(), (err, tol.max())


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [1e-45, 1e-38, 2.0 ** -100, 2.0 ** -30, 2.0 ** 100, 2.0 ** 127])
@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
def test_scales_of_any_size(dtype, scale, new):
    """Whole scores 0 .. 3: means of V where the scale leaves them equal, of V at the largest score where it does not."""
    s = px.GivenStep([500, 20], [new, 1], 16, 2, 2, 64, dtype, SEED + 3)
    s.give_q(1.0)
    for b, n in enumerate(s.lens):
        k = np.zeros((int(n), 2, 64))
        k[:, :, 7] = np.random.default_rng(b).integers(0, 4, (int(n), 2))
        s.give(b, k)
    s.check_exact(s.upload().attention(scale=scale), scale, 600)
