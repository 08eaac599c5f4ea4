"""More refusals of the paged-cache entry points, without a GPU."""
import numpy as np
import pytest

import arcllm_amd as arc
import paged_exact as px
import paged_lib as pl

A = 0x10000  # an address that is never followed: every call here is refused first, or has nothing to do


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_a_scale_whose_powers_of_two_pass_fp32_is_refused(sign):
    """scale log2 e is what the kernels multiply by: 2^127 is the last power of two that fits."""
    pages = arc.KvPages(A, 2 * A, 8, 16, 2)
    batch = arc.PagedBatch(2, 0, 4, 4, A, A, A)

    def call(scale):
        arc.paged_attention(pages, batch, A, 512, 2, 8 * A, 512, 4 * A, scale=sign * scale)

    call(2.0 ** 127)
    for scale in (3e38, float(np.finfo(np.float32).max)):
        with pytest.raises(arc.ArcError) as e:
            call(scale)
        assert e.value.code == 1 and "scale" in str(e.value)


@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16])
@pytest.mark.parametrize("course", ["equal", "rising", "falling"])
@pytest.mark.parametrize("case", px.CODED, ids=str)
def test_coded_rows_show_a_unit_left_out_or_taken_twice(case, course, dtype):
    """Of the longest row of each long context: without any 32 positions of one unit, or with them twice, an output
    leaves its bound (units of which 16 positions or more are seen)."""
    old, new, _, _, dim, window, sinks = case
    b = int(np.argmax(np.add(old, new)))
    n = old[b] + new[b]
    see = pl.visible(n - 1, n, window, sinks)
    K, V = (t[:, 0] for t in px.coded_rows(n, 1, dim, course))
    ref, tol = px.exact_row(np.ones((1, dim)), K[see], V[see], dim ** -0.5, n // 16, dtype)
    w = np.where(see, np.exp((K[:, 0] - K[see, 0].max()) * dim ** -0.5), 0.0)
    units = -(-n // 32)
    own = np.zeros((units, dim))
    np.add.at(own, (np.arange(n) // 32, V.argmax(1)), w)
    share = own.sum(1, keepdims=True)
    total, sums = w.sum(), own.sum(0)
    for sign in (-1, 1):
        off = np.abs((sums + sign * own) / (total + sign * share) - ref) / tol
        missed = (off.max(1) <= 1) & (np.add.reduceat(see, np.arange(0, n, 32), dtype=int) >= 16)
        assert not missed.any(), (sign, int(missed.sum()), off.max(1)[missed].min())
