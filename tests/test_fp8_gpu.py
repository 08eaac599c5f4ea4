"""The 8-bit block products on the GPU: quantisation bit for bit, products against float64 within their roundings."""
import numpy as np
import pytest
import torch

import arcllm_amd as arc
import fp8_lib as fl
import paged_lib as pl

pytestmark = pytest.mark.gpu

SEED = 0xF8
D = arc.DeviceBuffer.from_array
ALL = [arc.F32, arc.F16, arc.BF16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


def rng_of(*key):
    return np.random.default_rng([SEED, *key])


# ----------------------------------------------------------------- quantise
def run_quantize(x, dtype, ldx_pad=0, ldq_pad=0, lds_pad=0, stream=None):
    rows, cols = x.shape
    bits = fl.to_device_bits(x, dtype)
    nan = np.float32(np.nan) if dtype == arc.F32 else np.uint16(0x7FC0)
    padded = np.full((rows, cols + ldx_pad), nan, bits.dtype)
    padded[:, :cols] = bits
    dx = D(padded)
    q = D(np.full((rows, cols + ldq_pad), 0xA5, np.uint8))
    s = D(np.full((fl.blocks(cols), rows + lds_pad), -3.0, np.float32))
    arc.fp8_quantize(dtype, dx, cols + ldx_pad, arc.Fp8Rows(q, s, rows, cols, cols + ldq_pad, rows + lds_pad), stream=stream)
    if stream is not None:
        stream.synchronize()
    got_q, got_s = q.download(np.uint8).reshape(rows, -1), s.download(np.float32).reshape(fl.blocks(cols), -1)
    assert np.all(got_q[:, cols:] == 0xA5) and np.all(got_s[:, rows:] == -3.0)
    want_q, want_s = fl.quantize(fl.from_device_bits(bits, dtype).astype(np.float32))
    assert np.array_equal(got_s[:, :rows], want_s, equal_nan=True)
    dead = np.isnan(np.repeat(want_s.T, fl.BLOCK, 1)[:, :cols])  # any NaN will do there
    assert np.array_equal(got_q[:, :cols][~dead], want_q[~dead])
    assert np.all((got_q[:, :cols][dead] & 127) == 127)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (2, 112), (3, 144), (31, 512), (32, 528), (33, 496), (5, 3584), (70, 1040), (129, 272)])
def test_quantize(rows, cols, dtype):
    x = rng_of(rows, cols).standard_normal((rows, cols)) * np.exp(rng_of(rows).normal(0, 3, (rows, 1)))
    run_quantize(x, dtype)


@pytest.mark.parametrize("dtype", ALL)
def test_quantize_strides(dtype):
    run_quantize(rng_of(1).standard_normal((37, 400)), dtype, ldx_pad=24, ldq_pad=48, lds_pad=5)


@pytest.mark.parametrize("dtype", ALL)
def test_quantize_special_values(dtype):
    x = rng_of(2).standard_normal((16, 256)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2, :128] = 0.0
    x[3, 5], x[4, 200], x[5, 130] = np.inf, np.nan, -np.inf
    x[6] *= 2.0 ** -14
    x[7] *= 2.0 ** -24  # below fp16's range, or its last bits
    x[8] = 448.0 * np.where(np.arange(256) % 2, 1, -1)
    x[9] = np.linspace(-448, 448, 256)  # scale 1 or a little less: quotients next to the borders
    x[10, ::7] = 0.0
    run_quantize(x, dtype)


@pytest.mark.parametrize("dtype", [arc.F32, arc.BF16])
def test_quantize_far_ends_of_the_range(dtype):
    x = rng_of(3).standard_normal((12, 256)).astype(np.float32)
    for i, e in enumerate((-149, -140, -133, -126, -120, -100, -70, -60, 60, 100, 120, 125)):
        x[i] = np.ldexp(x[i], e)
    run_quantize(x, dtype)


def test_quantize_ties():
    """Quotients that are borders of e4m3, and their neighbours."""
    mid = (fl.VALUE[1:127] + fl.VALUE[:126]) / 2
    for scale in (1.0, 2.0 ** -20, 2.0 ** 30):
        x = np.zeros((3, 256), np.float32)
        x[:, 0] = x[:, 128] = 448.0  # scale 1
        x[0, 1:127] = mid
        x[1, 1:127] = np.nextafter(mid.astype(np.float32), np.float32(np.inf))
        x[2, 129:255] = -np.nextafter(mid.astype(np.float32), np.float32(0))
        run_quantize(x * np.float32(scale), arc.F32)


def test_quantize_many_rows():
    run_quantize(rng_of(4).standard_normal((70000, 16)), arc.F16)


@pytest.mark.parametrize("dtype", ALL)
def test_quantize_rows_at_any_16_bytes(dtype):
    """x at an odd multiple of 16 bytes, q and the scales too; rows 8 columns from the next."""
    rows, cols = 35, 272
    x = rng_of(5).standard_normal((rows, cols))
    bits = fl.to_device_bits(x, dtype)
    lead, size = 16 // bits.itemsize, (cols + 8) * rows
    flat = np.zeros(lead + size, bits.dtype)
    flat[lead:].reshape(rows, cols + 8)[:, :cols] = bits
    dx, q, s = D(flat), D(np.full(16 + rows * cols, 0xA5, np.uint8)), D(np.full(1 + 3 * rows, -3.0, np.float32))
    arc.fp8_quantize(dtype, dx.ptr + 16, cols + 8, arc.Fp8Rows(q.ptr + 16, s.ptr + 4, rows, cols))
    want_q, want_s = fl.quantize(fl.from_device_bits(bits, dtype).astype(np.float32))
    got_q, got_s = q.download(np.uint8), s.download(np.float32)
    assert np.all(got_q[:16] == 0xA5) and np.array_equal(got_q[16:].reshape(rows, cols), want_q)
    assert got_s[0] == -3.0 and np.array_equal(got_s[1:].reshape(3, rows), want_s)


# ------------------------------------------------------------------ product
class Product:
    def __init__(self, M, N, K, seed=0, mats=1, ldq_pad=0, lds_pad=0, ldw_pad=0, ldws_pad=0):
        rng = rng_of(M, N, K, seed)
        self.M, self.N, self.K = M, N, K
        self.xq, xs = fl.quantize(rng.standard_normal((M, K)) * np.exp(rng.normal(0, 1, (M, 1))))
        self.xs = xs
        self.w = [fl.weights(rng, N, K) for _ in range(mats)]
        # what lies between the rows: NaN
        def pad(a, n, fill):
            out = np.full((a.shape[0], a.shape[1] + n), fill, a.dtype)
            out[:, : a.shape[1]] = a
            return D(out)
        self.x = arc.Fp8Rows(pad(self.xq, ldq_pad, 0x7F), pad(xs, lds_pad, np.nan), M, K, K + ldq_pad, M + lds_pad)
        self.dw = [arc.Fp8Weights(pad(w, ldw_pad, 0x7F), pad(s, ldws_pad, np.nan), N, K, K + ldw_pad, fl.blocks(K) + ldws_pad)
                   for w, s in self.w]
        self.rng = rng

    def run(self, dtype, residual=False, in_place=False, ldy_pad=0, shift=0, stream=None, check=True):
        """y's rows `shift` elements behind a 256-byte border; what is not y stays as it was."""
        M, N, ldy = self.M, self.N, self.N + ldy_pad
        mark = np.float32(-77.0) if dtype == arc.F32 else np.uint16(0xABCD)
        flat = np.full(shift + M * ldy + 64, mark)
        size = flat.itemsize
        res = None
        if residual:
            res = fl.to_device_bits(self.rng.standard_normal((M, ldy)) * 30, dtype)
            if in_place:
                flat[shift: shift + M * ldy] = res.reshape(-1)
        y = D(flat)
        r = y.ptr + shift * size if in_place else D(np.concatenate([np.zeros(shift, flat.dtype), res.reshape(-1)])) if residual else None
        at = r.ptr + shift * size if residual and not in_place else r
        gated = len(self.dw) == 2
        ws = arc.DeviceBuffer(arc.fp8_gemm_workspace_bytes(N, self.K, M, gated))
        ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
        if gated:
            arc.fp8_gateup(*self.dw, self.x, dtype, y.ptr + shift * size, ldy, ws, stream=stream)
        else:
            arc.fp8_gemm(self.dw[0], self.x, dtype, y.ptr + shift * size, ldy, ws, residual=at, ldr=ldy, stream=stream)
        if stream is not None:
            stream.synchronize()
        out = y.download(flat.dtype)
        assert np.array_equal(out[:shift], flat[:shift]) and np.array_equal(out[shift + M * ldy:], flat[shift + M * ldy:])
        rows = out[shift: shift + M * ldy].reshape(M, ldy)
        before = flat[shift: shift + M * ldy].reshape(M, ldy)
        assert np.array_equal(rows[:, N:], before[:, N:]), "columns behind y"
        got = fl.from_device_bits(rows[:, :N], dtype)
        if check:
            self.check(got, dtype, None if res is None else fl.from_device_bits(res[:, :N], dtype))
        return got

    def check(self, got, dtype, res=None):
        parts = [fl.product(self.xq, self.xs, w, s, dtype) for w, s in self.w]
        y, tol = parts[0]
        if len(parts) == 2:
            y, tol = fl.gated(*parts[0], *parts[1], dtype)
        if res is not None:
            y, tol = y + res, tol + np.abs(y + res) * 2.0 ** -24
        fl.near(got, y, tol, dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 129])
def test_rows(M, dtype):
    Product(M, 200, 384).run(dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("N", [1, 3, 15, 16, 17, 64, 127, 128, 129, 255, 257, 300])
@pytest.mark.parametrize("M", [3, 20, 50, 90])
def test_outputs(M, N, dtype):
    Product(M, N, 256).run(dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("K", [16, 32, 64, 80, 112, 128, 144, 192, 240, 256, 272, 400, 1040])
@pytest.mark.parametrize("M", [5, 30, 60, 100])
def test_depths(M, K, dtype):
    Product(M, 130, K).run(dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("M,N,K", [(1, 40, 128), (16, 130, 272), (20, 64, 384), (33, 190, 256), (64, 129, 1040), (100, 70, 128), (130, 333, 512),
                                   (200, 128, 640), (70, 31, 48)])
def test_gated(M, N, K, dtype):
    Product(M, N, K, mats=2).run(dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("M,N,K,pad,shift", [(1, 64, 256, 0, 0), (7, 33, 144, 7, 1), (20, 130, 256, 2, 3), (40, 128, 384, 8, 0), (70, 129, 256, 0, 1),
                                             (130, 256, 512, 4, 4)])
def test_residual(M, N, K, pad, shift, in_place, dtype):
    Product(M, N, K).run(dtype, residual=True, in_place=in_place, ldy_pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("mats", [1, 2])
@pytest.mark.parametrize("M", [4, 30, 60, 140])
def test_strides(M, mats, dtype):
    Product(M, 150, 272, mats=mats, ldq_pad=32, lds_pad=3, ldw_pad=16, ldws_pad=2).run(dtype, ldy_pad=5, shift=2)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("M,N,K", [(20, 100, 4096), (60, 130, 3000 // 16 * 16), (130, 260, 4096), (300, 100, 8192), (129, 128, 2048 + 16)])
def test_blocks_in_several_parts(M, N, K, dtype):
    Product(M, N, K).run(dtype, residual=True)


@pytest.mark.parametrize("K", [4096, 2000])
def test_gated_in_several_parts(K):
    Product(100, 90, K, mats=2).run(arc.BF16)
    Product(30, 90, K, mats=2).run(arc.F32)


def reference(p, dtype=torch.float64):
    """The products in float64 by torch on the GPU."""
    ys = []
    x = torch.from_numpy(fl.VALUE[p.xq] * fl.spread(p.xs.T.astype(np.float64), p.M, p.K)).cuda()
    for w, s in p.w:
        ys.append(x @ torch.from_numpy(fl.VALUE[w] * fl.spread(s.astype(np.float64), p.N, p.K)).cuda().t().contiguous())
    size = x.abs().amax()
    return ys, size


@pytest.mark.parametrize("dtype", [arc.F16, arc.BF16, arc.F32])
@pytest.mark.parametrize("M,N,K,mats", [(700, 3000, 384, 1), (1030, 6200, 256, 1), (600, 5100, 384, 2), (2100, 2000, 128, 1), (257, 9000, 640, 2),
                                        (900, 1500, 2048, 1)])
def test_large(M, N, K, mats, dtype):
    """Tiles of every size, more of them than workgroups, edges in both directions: relative to the rows' size."""
    p = Product(M, N, K, mats=mats)
    got = p.run(dtype, check=False)
    ys, _ = reference(p)
    y = (ys[0] * torch.sigmoid(ys[0]) * ys[1] if mats == 2 else ys[0]).cpu().numpy()
    # sums of absolute values: |x| |w|^T
    a = [torch.from_numpy(np.abs(fl.VALUE[p.xq]) * fl.spread(p.xs.T.astype(np.float64), M, K)).cuda()
         @ torch.from_numpy(np.abs(fl.VALUE[w]) * fl.spread(s.astype(np.float64), N, K)).cuda().t().contiguous() for w, s in p.w]
    # of 8 products the largest is at most their sum: 7 * 2^-13 of the sum of absolute values; fp32 as in fp8_lib.product
    rel = (fl.BLOCK + fl.blocks(K) + 4) * 2.0 ** -23 + (0 if dtype == arc.F32 else 7 * 2.0 ** -13)
    d = [(t * rel).cpu().numpy() for t in a]
    tol = d[0] if mats == 1 else fl.gated(ys[0].cpu().numpy(), d[0], ys[1].cpu().numpy(), d[1], dtype)[1]
    fin = fl.near(got, y, tol, dtype)
    # and on the whole no further off than the type's rounding and a little of the cores' own
    off = np.linalg.norm((got - y)[fin]) / np.linalg.norm(y[fin])
    assert off <= {arc.F32: 2e-6, arc.F16: 2.0 ** -11, arc.BF16: 2.0 ** -8}[dtype], off


def test_rows_alone_have_nan():
    """A NaN in x or its scale is its row's, one in w its output's."""
    p = Product(70, 100, 256)
    base = p.run(arc.F32)
    q, s = p.xq.copy(), p.xs.copy()
    q[5, 7], s[1, 9] = 0x7F, np.nan
    w, ws = p.w[0][0].copy(), p.w[0][1]
    w[11, 200] = 0xFF
    p.x = arc.Fp8Rows(D(q), D(s), 70, 256)
    p.dw = [arc.Fp8Weights(D(w), D(ws), 100, 256)]
    for dtype in ALL:
        got = p.run(dtype, check=False)
        nan = np.zeros((70, 100), bool)
        nan[[5, 9]] = True
        nan[:, 11] = True
        assert np.array_equal(np.isnan(got), nan)
        if dtype == arc.F32:
            assert np.array_equal(got[~nan], base[~nan])


@pytest.mark.parametrize("K", [144, 272])
@pytest.mark.parametrize("M", [10, 40, 80])
def test_a_nan_behind_the_last_column_is_not_read(M, K):
    """K ends inside a block, and what lies behind it in the row is NaN (test_strides) or the next row."""
    p = Product(M, 40, K)
    for dtype in ALL:
        p.run(dtype)


def test_huge_and_tiny_scales():
    p = Product(20, 40, 256)
    for e in (-60, 55):
        q = Product(20, 40, 256)
        q.xs = np.ldexp(p.xs, e).astype(np.float32)
        q.x = arc.Fp8Rows(D(q.xq), D(q.xs), 20, 256)
        q.run(arc.F32)


@pytest.mark.parametrize("M", [3, 40, 300])
def test_same_call_twice_gives_the_same_bits(M):
    p = Product(M, 300, 4096)
    for dtype in (arc.F32, arc.BF16):
        assert np.array_equal(p.run(dtype, check=False), p.run(dtype, check=False))


def test_calls_on_their_own_streams():
    ps = [Product(M, 200, 2048, seed=i) for i, M in enumerate((5, 60, 200))]
    streams = [arc.Stream() for _ in ps]
    for p, s in zip(ps, streams):
        p.run(arc.F16, stream=s)


def test_weights_past_32_bits():
    """Rows of w 2^32 bytes and more behind its first."""
    K, N = 16, 1100
    ld = 1 << 22
    w = torch.zeros(N * ld, dtype=torch.uint8, device="cuda")
    p = Product(40, N, K)
    rows = w.view(N, ld)
    rows[:, :K] = torch.from_numpy(p.w[0][0]).cuda()
    torch.cuda.synchronize()
    p.dw = [arc.Fp8Weights(w.data_ptr(), D(p.w[0][1]), N, K, ld)]
    for M in (40, 4):
        q = Product(M, N, K)
        q.w, q.dw = p.w, p.dw
        for dtype in (arc.F32, arc.BF16):
            q.run(dtype)


@pytest.mark.parametrize("M,N,K,mats", [(2100, 20000, 256, 2), (1900, 30001, 128, 1), (1000, 3584, 8192, 1), (2048, 3584, 4096, 1), (1100, 1800, 8192, 2)])
def test_more_tiles_than_the_card_holds(M, N, K, mats):
    """Workgroups that go on to a second and third tile, and large tiles in parts; compared on the GPU, with the sum of
    absolute values as in test_large."""
    g = torch.Generator(device="cuda").manual_seed(SEED)
    value = torch.from_numpy(fl.VALUE).cuda()
    def codes(n):
        c = torch.randint(0, 256, (n, K), generator=g, device="cuda", dtype=torch.uint8)
        return torch.where((c & 127) == 127, 3, c)
    x, xs = codes(M), torch.rand(fl.blocks(K), M, generator=g, device="cuda") + 0.1
    ws = [(codes(N), torch.rand(fl.blocks(N), fl.blocks(K), generator=g, device="cuda") * 1e-3 + 1e-4) for _ in range(mats)]
    y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    space = torch.full((arc.fp8_gemm_workspace_bytes(N, K, M, mats == 2),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dx = arc.Fp8Rows(x.data_ptr(), xs.data_ptr(), M, K)
    dw = [arc.Fp8Weights(w.data_ptr(), s.data_ptr(), N, K) for w, s in ws]
    args = (dx, arc.BF16, y.data_ptr(), N, space.data_ptr())
    arc.fp8_gateup(*dw, *args) if mats == 2 else arc.fp8_gemm(*dw, *args)
    arc.synchronize()
    sums, sizes = [], []
    for f, out in ((lambda t: t, sums), (torch.abs, sizes)):
        a = f(value[x.long()]) * xs.t().double().repeat_interleave(128, 1)[:, :K]
        for w, s in ws:
            b = f(value[w.long()]) * s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
            out.append(a @ b.t().contiguous())
    d = [t * ((fl.BLOCK + fl.blocks(K) + 4) * 2.0 ** -23 + 7 * 2.0 ** -13) for t in sizes]
    want, tol = sums[0], d[0]
    if mats == 2:  # as fp8_lib.gated
        gate = sums[0] * torch.sigmoid(sums[0])
        want = gate * sums[1]
        tol = 1.1 * d[0] * (sums[1].abs() + d[1]) + gate.abs() * d[1] + want.abs() * (2.0 ** -20 + sums[0].abs() * 2.0 ** -22)
    tol = tol + (want.abs() + tol) * 2.0 ** -8 * 1.01 + 2.0 ** -120
    assert bool(torch.isfinite(y).all())
    assert bool(((y.double() - want).abs() <= tol).all())
    assert float((y.double() - want).norm() / want.norm()) <= 2.0 ** -8
