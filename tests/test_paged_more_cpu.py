"""More refusals of the paged-cache entry points, without a GPU."""
import numpy as np
import pytest

import arcllm_amd as arc

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
