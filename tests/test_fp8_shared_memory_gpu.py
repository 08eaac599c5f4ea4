"""One buffer whose rows hold an input row, its values in 8 bits, a row of scales, and an output row, side by side: the
arrays of a call share no byte, so the calls take it."""
import numpy as np
import pytest

import arcllm_amd as arc
import fp8_lib as fl

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


@pytest.mark.parametrize("M", [4, 20, 70])
def test_rows_side_by_side(M):
    rng = np.random.default_rng([0xF8, M])
    N, K = 130, 272
    x = rng.standard_normal((M, K)).astype(np.float32)
    wq, ws = fl.weights(rng, N, K)
    at_q, at_s, at_y = 4 * K, 5 * K, 5 * K + 4 * 80
    stride = (at_y + 4 * N + 31) // 32 * 32
    host = np.full((M, stride), 0xA5, np.uint8)
    host[:, : 4 * K] = x.view(np.uint8)
    buf = arc.DeviceBuffer.from_array(host)
    rows = arc.Fp8Rows(buf.ptr + at_q, buf.ptr + at_s, M, K, stride, stride // 4)
    arc.fp8_quantize(arc.F32, buf.ptr, stride // 4, rows)
    w = arc.Fp8Weights(arc.DeviceBuffer.from_array(wq), arc.DeviceBuffer.from_array(ws), N, K)
    space = arc.DeviceBuffer(arc.fp8_gemm_workspace_bytes(N, K, M))
    arc.fp8_gemm(w, rows, arc.F32, buf.ptr + at_y, stride // 4, space)
    got = buf.download(np.uint8).reshape(M, stride)
    q, s = fl.quantize(x)
    assert np.array_equal(got[:, at_q: at_q + K], q)
    blocks = fl.blocks(K)
    assert np.array_equal(got[:blocks, at_s: at_s + 4 * M].copy().view(np.float32), s)
    assert np.all(got[blocks:, at_s: at_s + 4 * M] == 0xA5) and np.array_equal(got[:, : 4 * K], host[:, : 4 * K])
    fl.near(got[:, at_y: at_y + 4 * N].copy().view(np.float32).astype(np.float64), *fl.product(q, s, wq, ws, arc.F32), arc.F32)
