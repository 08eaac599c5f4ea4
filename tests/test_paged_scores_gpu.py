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
