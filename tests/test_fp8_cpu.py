"""The 8-bit block products without a GPU: refusals before any launch, and the oracle's rounding."""
import ctypes as C

import numpy as np
import pytest

import arcllm_amd as arc
import fp8_lib as fl

A = 0x100000  # an address that is never followed


def rows(**over):
    d = dict(q=A, scales=2 * A, rows=40, cols=256)
    d.update(over)
    return arc.Fp8Rows(**d)


def weights(**over):
    d = dict(w=4 * A, scales=5 * A, rows=300, cols=256)
    d.update(over)
    return arc.Fp8Weights(**d)


def refused(fn):
    with pytest.raises(arc.ArcError) as e:
        fn()
    assert e.value.code in (1, 2) and len(str(e.value)) > 20


def quantize(out=None, dtype=arc.F32, x=8 * A, ldx=256):
    arc.fp8_quantize(dtype, x, ldx, out or rows())


def gemm(w=None, x=None, dtype=arc.F32, y=8 * A, ldy=300, ws=16 * A, **kw):
    arc.fp8_gemm(w or weights(), x or rows(), dtype, y, ldy, ws, **kw)


def gateup(g=None, u=None, x=None, dtype=arc.F32, y=8 * A, ldy=300, ws=16 * A):
    arc.fp8_gateup(g or weights(), u or weights(), x or rows(), dtype, y, ldy, ws)


BAD_ROWS = [dict(q=None), dict(scales=None), dict(cols=0), dict(cols=250), dict(ldq=240), dict(ldq=264), dict(lds=39),
            dict(q=A + 8), dict(scales=2 * A + 2), dict(rows=(1 << 24) + 1), dict(cols=(1 << 22) + 16, ldq=(1 << 22) + 16),
            dict(ldq=1 << 23)]


@pytest.mark.parametrize("over", BAD_ROWS, ids=str)
def test_bad_rows(over):
    refused(lambda: quantize(rows(**over), ldx=1 << 23))
    refused(lambda: gemm(x=rows(**over)))


@pytest.mark.parametrize("over", [dict(w=None), dict(scales=None), dict(rows=0), dict(cols=128), dict(ldw=128), dict(lds=1),
                                  dict(w=4 * A + 4), dict(rows=(1 << 24) + 1)], ids=str)
def test_bad_weights(over):
    refused(lambda: gemm(weights(**over)))
    refused(lambda: gateup(g=weights(**over)))
    refused(lambda: gateup(u=weights(**over)))


@pytest.mark.parametrize("call", [
    lambda: quantize(dtype=7), lambda: quantize(x=None), lambda: quantize(x=8 * A + 4), lambda: quantize(ldx=248),
    lambda: quantize(ldx=260), lambda: quantize(x=A + 512),  # over its own rows
    lambda: gemm(dtype=8), lambda: gemm(y=None), lambda: gemm(ws=None), lambda: gemm(ws=16 * A + 16), lambda: gemm(ldy=299),
    lambda: gemm(y=8 * A + 2), lambda: gemm(residual=9 * A, ldr=299), lambda: gemm(residual=9 * A + 1, ldr=300),
    lambda: gemm(residual=8 * A + 40, ldr=300), lambda: gemm(residual=8 * A, ldr=304), lambda: gemm(y=A + 1024),
    lambda: gateup(u=weights(rows=301)), lambda: gateup(dtype=3), lambda: gateup(ldy=10),
    lambda: gemm(weights(rows=1 << 24, cols=16), rows(rows=1 << 24, cols=16), y=1 << 50, ldy=1 << 24),  # more tiles than a call takes
])
def test_refusals(call):
    refused(call)


def test_nothing_to_do():
    quantize(rows(rows=0))
    gemm(x=rows(rows=0))
    gateup(x=rows(rows=0))


def test_null_structs():
    L = arc.lib()
    x, w = rows(), weights()
    assert L.arc_fp8_quantize(0, A, 256, None, None) == 1
    assert L.arc_fp8_gemm(None, C.byref(x), 0, A, 300, None, 0, A, None) == 1
    assert L.arc_fp8_gemm(C.byref(w), None, 0, A, 300, None, 0, A, None) == 1
    assert L.arc_fp8_gateup(C.byref(w), None, C.byref(x), 0, 8 * A, 300, 16 * A, None) == 1


def test_workspace_sizes():
    for bad in ((0, 256, 4), (300, 0, 4), (300, 250, 4), (300, (1 << 22) + 16, 4), ((1 << 24) + 1, 256, 4), (300, 256, (1 << 24) + 1)):
        refused(lambda: arc.fp8_gemm_workspace_bytes(*bad))
    assert arc.fp8_gemm_workspace_bytes(300, 256, 0) >= 256
    # 45 rows need no parts' sums since k_fp8_own takes them; 128 rows do
    assert arc.fp8_gemm_workspace_bytes(3584, 18944, 45) >= arc.fp8_gemm_workspace_bytes(3584, 18944, 4)
    assert arc.fp8_gemm_workspace_bytes(3584, 18944, 128) >= 2 * 128 * 3584 * 4


def test_oracle_rounding():
    v = fl.VALUE[:127]
    assert np.array_equal(fl.encode(v), np.arange(127)) and np.array_equal(fl.encode(-v[1:]), np.arange(1, 127) + 128)
    mid = (v[1:] + v[:-1]) / 2
    assert np.array_equal(fl.encode(mid) % 2, np.zeros(126))  # ties to even
    assert np.array_equal(fl.encode(np.nextafter(mid, 1e9)), np.arange(1, 127)) and np.array_equal(fl.encode(np.nextafter(mid, 0)), np.arange(126))
    assert fl.encode(448.00003) == 126 and fl.encode(-0.0) == 128
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(5).standard_normal(5000).astype(np.float32) * 90
    assert np.array_equal(fl.encode(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
