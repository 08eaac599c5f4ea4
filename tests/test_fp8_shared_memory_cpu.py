"""The 8-bit products refuse outputs that share memory with what a call reads or else writes, before any launch."""
import pytest

import arcllm_amd as arc

A = 0x1000000  # addresses that are never followed


def rows(**over):
    # 40 x 256: q [A, A + 0x2800), scales [2 A, 2 A + 0x140)
    return arc.Fp8Rows(**{**dict(q=A, scales=2 * A, rows=40, cols=256), **over})


def weights(n=0, **over):
    # 300 x 256: w [.., + 0x12c00), scales [.., + 0x18)
    return arc.Fp8Weights(**{**dict(w=(4 + n) * A, scales=(6 + n) * A, rows=300, cols=256), **over})


def refused(fn):
    with pytest.raises(arc.ArcError, match="share memory") as e:
        fn()
    assert e.value.code == 1


def quantize(x, out, dtype=arc.F32, ldx=256):
    arc.fp8_quantize(dtype, x, ldx, out)


@pytest.mark.parametrize("call", [
    lambda: quantize(8 * A, rows(scales=8 * A)),                      # x and scales
    lambda: quantize(8 * A, rows(scales=8 * A + 40 * 1024 - 4)),      # x's last value
    lambda: quantize(8 * A + 0x130, rows(scales=8 * A)),              # the last scales
    lambda: quantize(8 * A, rows(scales=A)), lambda: quantize(8 * A, rows(scales=A + 0x27FC)), lambda: quantize(8 * A, rows(q=2 * A + 0x130)),
    lambda: quantize(8 * A, rows(ldq=512, scales=A + 0x1F0)),         # begins in the gap of q's first row, reaches its second
], ids=list("abcdefg"))
def test_quantize(call):
    refused(call)


def gemm(y=8 * A, dtype=arc.F32, ldy=300, ws=16 * A, w=None, x=None, **kw):
    arc.fp8_gemm(w or weights(), x or rows(), dtype, y, ldy, ws, **kw)


def gateup(y=8 * A, dtype=arc.BF16, ldy=300, ws=16 * A, x=None):
    arc.fp8_gateup(weights(), weights(1), x or rows(), dtype, y, ldy, ws)


@pytest.mark.parametrize("y", [2 * A, 2 * A + 0x13C, 4 * A, 4 * A + 0x12BF8, 6 * A, 6 * A + 0x14], ids=hex)
def test_outputs(y):
    refused(lambda: gemm(y=y))
    refused(lambda: gateup(y=y))


@pytest.mark.parametrize("y", [5 * A, 5 * A + 0x12BF8, 7 * A, 7 * A + 0x14], ids=hex)
def test_outputs_over_the_up_weights(y):
    refused(lambda: gateup(y=y))


def test_outputs_between_rows():
    # scales in the gap behind y's rows of 1200 bytes: those that reach the next row
    refused(lambda: gemm(ldy=512, x=rows(scales=8 * A + 2048 - 4, lds=40)))


# 128 rows of 3584 x 18944 are cut in parts, whose sums go into the workspace
BIG_X, BIG_W = dict(rows=128, cols=18944), dict(rows=3584, cols=18944)


@pytest.mark.parametrize("ws", ["q", "scales", "w", "w_scales", "y", "residual"])
def test_workspace(ws):
    at = dict(q=1 << 32, scales=2 << 32, w=3 << 32, w_scales=4 << 32, y=5 << 32, residual=6 << 32)
    x = arc.Fp8Rows(at["q"], at["scales"], **BIG_X)
    w = arc.Fp8Weights(at["w"], at["w_scales"], **BIG_W)
    refused(lambda: arc.fp8_gemm(w, x, arc.F32, at["y"], 3584, at[ws], residual=at["residual"], ldr=3584))
    refused(lambda: arc.fp8_gemm(w, x, arc.F32, at["y"], 3584, at[ws] - 256, residual=at["residual"], ldr=3584))
