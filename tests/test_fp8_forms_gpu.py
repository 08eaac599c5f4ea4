"""Every kernel, tile and number of parts of the 8-bit products (fp8_forms.py) against float64, computed on the GPU: plain with and
without a residual, with the activation, in each type of output."""
import pytest
import torch

import arcllm_amd as arc
import fp8_forms as ff
import fp8_lib as fl

pytestmark = pytest.mark.gpu

TYPES = {arc.F32: torch.float32, arc.F16: torch.float16, arc.BF16: torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert arc.device_count() >= 1, "no HIP device visible"


class Product:
    """Random e4m3 numbers with scales of different size; sums in float64 and the sums of absolute values."""

    def __init__(self, M, N, K, gated, seed=0):
        g = torch.Generator(device="cuda").manual_seed(0xF8 + seed)
        self.M, self.N, self.K, self.gated = M, N, K, gated
        value = torch.from_numpy(fl.VALUE).cuda()

        def codes(n):
            c = torch.randint(0, 256, (n, K), generator=g, device="cuda", dtype=torch.uint8)
            return torch.where((c & 127) == 127, 3, c)

        rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
        self.x, self.xs = codes(M), rand(fl.blocks(K), M) + 0.1
        self.w = [(codes(N), rand(fl.blocks(N), fl.blocks(K)) * 4e-5 + 1e-5) for _ in range(1 + gated)]
        self.res = torch.randn(M, N, generator=g, device="cuda") * 3
        self.sums, self.sizes = [], []
        for f, out in ((lambda t: t, self.sums), (torch.abs, self.sizes)):
            a = f(value[self.x.long()]) * self.xs.t().double().repeat_interleave(128, 1)[:, :K]
            for w, s in self.w:
                b = f(value[w.long()]) * s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
                out.append(a @ b.t().contiguous())
        self.dx = arc.Fp8Rows(self.x.data_ptr(), self.xs.data_ptr(), M, K)
        self.dw = [arc.Fp8Weights(w.data_ptr(), s.data_ptr(), N, K) for w, s in self.w]
        self.space = torch.full((arc.fp8_gemm_workspace_bytes(N, K, M, bool(gated)),), 255, dtype=torch.uint8, device="cuda")

    def start(self, dtype, residual=False, ldy=None, stream=None):
        ldy = ldy or self.N
        y = torch.full((self.M, ldy), float("nan"), dtype=TYPES[dtype], device="cuda")
        res = None
        if residual:
            res = self.res.to(TYPES[dtype])
            torch.cuda.synchronize()
        torch.cuda.synchronize()
        self.call(dtype, y, res, stream)
        return y, res

    def call(self, dtype, y, res=None, stream=None):
        args = (self.dx, dtype, y.data_ptr(), y.shape[1], self.space.data_ptr())
        if self.gated:
            arc.fp8_gateup(*self.dw, *args, stream=stream)
        else:
            arc.fp8_gemm(*self.dw, *args, residual=None if res is None else res.data_ptr(), ldr=self.N, stream=stream)

    def check(self, dtype, y, res=None):
        # fp32's own (fp8_lib.product), and for 16 bits 7 * 2^-13 of each 8 products' largest, which is at most their sum
        rel = (fl.BLOCK + fl.blocks(self.K) + 4) * 2.0 ** -23 + (0 if dtype == arc.F32 else 7 * 2.0 ** -13)
        d = [t * rel for t in self.sizes]
        want, tol = self.sums[0], d[0]
        if self.gated:  # as fp8_lib.gated
            g, u = self.sums
            gate = g * torch.sigmoid(g)
            want = gate * u
            tol = 1.1 * d[0] * (u.abs() + d[1]) + gate.abs() * d[1] + want.abs() * (2.0 ** -20 + g.abs() * 2.0 ** -22)
        if res is not None:
            want = want + res.double()
            tol = tol + want.abs() * 2.0 ** -24
        half = fl.HALF_STEP[dtype]
        tol = tol + (want.abs() + tol) * half * 1.01 + (2.0 ** -25 if dtype == arc.F16 else 2.0 ** -120)
        got = y[:, : self.N].double()
        assert bool(torch.isfinite(got).all())
        off = (got - want).abs() / tol
        assert float(off.max()) <= 1.0, (float(off.max()), [int(i) for i in divmod(int(off.argmax()), self.N)])
        assert bool(torch.isnan(y[:, self.N:]).all()), "columns behind y"


def types(y16):
    return [arc.F16, arc.BF16] if y16 else [arc.F32]


@pytest.mark.parametrize("case", ff.ALL, ids=lambda c: f"{c[5]}-{'x'.join(map(str, c[:3]))}-{'gated' if c[3] else 'plain'}-{'y16' if c[4] else 'y32'}-{c[6]}")
def test_form(case):
    M, N, K, gated, y16, *_ = case
    p = Product(M, N, K, gated)
    for dtype in types(y16):
        y, _ = p.start(dtype)  # rows side by side: wide stores where N is a multiple of 4
        torch.cuda.synchronize()
        p.check(dtype, y)
        if not gated:
            y, res = p.start(dtype, residual=True)
            torch.cuda.synchronize()
            p.check(dtype, y, res)
    y, _ = p.start(types(y16)[-1], ldy=N + 3)  # narrow ones
    torch.cuda.synchronize()
    p.check(types(y16)[-1], y)


@pytest.mark.parametrize("y16", [0, 1])
def test_calls_under_way_together(y16):
    """Products of several forms, each on its own stream with its own workspace, several calls each, before any of them is waited for."""
    shapes = [(64, 9001, 640, 1), (128, 3584, 2048, 0), (300, 777, 640, 0), (45, 300, 1040, 0), (646, 13944, 640, 1)]
    ps = [Product(*s, seed=i) for i, s in enumerate(shapes)]
    dtype = types(y16)[-1]
    ys = [[torch.full((p.M, p.N), float("nan"), dtype=TYPES[dtype], device="cuda") for _ in range(4)] for p in ps]
    streams = [arc.Stream() for _ in ps]
    torch.cuda.synchronize()
    for i in range(4):
        for p, y, s in zip(ps, ys, streams):
            p.call(dtype, y[i], stream=s)
    for s in streams:
        s.synchronize()
    for p, y in zip(ps, ys):
        for t in y:
            p.check(dtype, t)
            assert torch.equal(t, y[0])


def test_captured_products_side_by_side():
    """Two graphs of products in parts, each with its own workspace, replayed at once; every replay equals the eager call."""

    class Here:
        def __init__(self, s):
            self.handle = s.cuda_stream

    ps = [Product(128, 3584, 2048, 0, seed=5), Product(64, 300, 4096, 1, seed=6)]
    want, ys, graphs = [], [], []
    for p in ps:
        y = torch.zeros(p.M, p.N, device="cuda")
        p.call(arc.F32, y)
        torch.cuda.synchronize()
        want.append(y.clone())
        p.check(arc.F32, y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.call(arc.F32, y, stream=Here(torch.cuda.current_stream()))
        graphs.append(graph)
        ys.append(y)
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(4):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for y, w in zip(ys, want):
            assert torch.equal(y, w)
