"""Float64 statements of the paged-cache entry points, and random serving steps to
hold them to: the plan in plain Python, rotary positions in extended precision,
attention row by row."""
import numpy as np

import arcllm_amd as arc

HALF_STEP = {arc.F16: 2.0 ** -11, arc.BF16: 2.0 ** -8}  # finfo.eps / 2


# ------------------------------------------------------------- 16-bit types
def to_bits(x, dtype):
    """float array -> the bits of its values rounded to nearest even, uint16."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == arc.F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    r[np.isnan(x)] = 0x7FC0
    return r


def from_bits(b, dtype):
    b = np.ascontiguousarray(b, np.uint16)
    if dtype == arc.F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


# --------------------------------------------------------------------- plan
def pages_of(n, page):
    return -(-n // page)


def plan(old, new, page, tables, max_pages, rows, max_new, stack, count, num_pages):
    """What arc_paged_plan leaves: dict of tables, lens, starts, positions, slots, stack, count, status."""
    B = len(old)
    tables, stack = tables.copy(), stack.copy()
    refuse = 0
    fresh = [0 if n == arc.PAGED_RELEASE else n for n in new]
    for o, n in zip(old, new):
        if n != arc.PAGED_RELEASE and n > max_new:
            refuse |= arc.PLAN_MAX_NEW
        if o + (0 if n == arc.PAGED_RELEASE else n) > min(max_pages * page, 2 ** 31 - 1):
            refuse |= arc.PLAN_TABLE
    lacking = 0
    if not refuse:
        back = sum(pages_of(o, page) for o, n in zip(old, new) if n == arc.PAGED_RELEASE)
        take = sum(pages_of(o + n, page) - pages_of(o, page) for o, n in zip(old, new) if n != arc.PAGED_RELEASE)
        if sum(fresh) > rows:
            refuse |= arc.PLAN_TOKENS
        if count + back > num_pages:
            refuse |= arc.PLAN_FREE_LIST
        elif take > count + back:
            refuse |= arc.PLAN_NO_PAGES
            lacking = take - count - back
    positions, slots = np.zeros(rows, np.uint32), np.full(rows, arc.NO_SLOT, np.uint32)
    if refuse:
        return dict(tables=tables, lens=np.array(old, np.uint32), starts=np.zeros(B + 1, np.uint32),
                    positions=positions, slots=slots, stack=stack, count=count,
                    status=np.array([refuse, lacking, 0, 0], np.uint32))
    for b in range(B):
        if new[b] == arc.PAGED_RELEASE:
            for i in range(pages_of(old[b], page)):
                stack[count] = tables[b, i]
                count += 1
    popped, starts, n = 0, [0], 0
    for b in range(B):
        if new[b] != arc.PAGED_RELEASE:
            for i in range(pages_of(old[b], page), pages_of(old[b] + new[b], page)):
                count -= 1
                popped += 1
                tables[b, i] = stack[count]
            for p in range(old[b], old[b] + new[b]):
                positions[n] = p
                slots[n] = tables[b, p // page] * page + p % page
                n += 1
        starts.append(n)
    lens = [0 if w == arc.PAGED_RELEASE else o + w for o, w in zip(old, new)]
    return dict(tables=tables, lens=np.array(lens, np.uint32), starts=np.array(starts, np.uint32), positions=positions,
                slots=slots, stack=stack, count=count, status=np.array([0, 0, n, popped], np.uint32))


# --------------------------------------------------------------------- rope
def rope_freqs(rot, theta, scaling=arc.ROPE_PLAIN, factor=1.0, original_ctx=0, beta_fast=32.0, beta_slow=1.0,
               freq_factors=None):
    """(angles per position, extended precision; factor on the rotated values)."""
    L = np.longdouble
    i = np.arange(rot // 2, dtype=L)
    f = L(theta) ** (-2 * i / L(rot))
    scale = 1.0
    if scaling == arc.ROPE_LINEAR:
        f = f / L(factor)
    if scaling == arc.ROPE_YARN:
        def at(beta):
            return rot * np.log(original_ctx / (beta * 2 * np.pi)) / (2 * np.log(theta))
        low, high = max(np.floor(at(beta_fast)), 0), min(np.ceil(at(beta_slow)), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f = f * (1 - ramp) + f / L(factor) * ramp
        scale = 0.1 * np.log(factor) + 1.0
    if freq_factors is not None:
        f = f / np.asarray(freq_factors, np.float32).astype(L)
    return f, scale


def rotate(x, positions, freqs, scale, layout):
    """x [N, heads, D] float64 rotated at positions [N]; also |a| + |b| of each value's pair (times scale),
    what errors of the angle are multiplied by."""
    n = len(freqs)
    angle = positions.astype(np.longdouble)[:, None] * freqs[None, :]
    c, s = np.cos(angle).astype(np.float64)[:, None, :], np.sin(angle).astype(np.float64)[:, None, :]
    i = np.arange(n) * (1 if layout == arc.ROPE_HALF else 2)
    j = i + (n if layout == arc.ROPE_HALF else 1)
    a, b = x[..., i], x[..., j]
    y, size = x.copy(), np.zeros_like(x)
    y[..., i], y[..., j] = (a * c - b * s) * scale, (a * s + b * c) * scale
    size[..., i] = size[..., j] = (np.abs(a) + np.abs(b)) * scale
    return y, size


# ---------------------------------------------------------------- attention
def visible(pos, length, window, sinks):
    j = np.arange(length)
    see = j <= pos
    return see & ((pos - j < window) | (j < sinks)) if window else see


def attend(q, K, V, pos, scale, window=0, sinks=0, dropped=None):
    """One row: q [heads, D]; K, V [length, kv_heads, D] float64 (only visible rows are read).  Returns the
    row's output [heads, D], sum_j p_j |v_j|, the largest rounding of a score in fp32 (D + 2 roundings of
    sum |q k|) and the number of positions it sees."""
    see = visible(pos, len(K), window, sinks)
    if dropped is not None:
        see &= ~dropped
    heads, D = q.shape
    hpk = heads // K.shape[1]
    if not see.any():
        return np.zeros_like(q), np.zeros_like(q), 0.0, 0
    k, v = K[see].repeat(hpk, 1), V[see].repeat(hpk, 1)
    s = np.einsum("hd,jhd->hj", q, k) * scale
    off = np.einsum("hd,jhd->hj", np.abs(q), np.abs(k)).max() * scale * (D + 2) * 2.0 ** -24
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return np.einsum("hj,jhd->hd", p, v), np.einsum("hj,jhd->hd", p, np.abs(v)), off, int(see.sum())


def attention_bound(ref, mass, off, seen, vmax, dtype):
    """How far one element may be off: the output's rounding; the weights' rounding to the type, the scores'
    rounding in both a weight and the sum of weights, exp2's argument and result (2^-20), sums of `seen`
    terms in fp32, each times sum p |v|; fp16 weights below its normal range round by 2^-25 of the largest."""
    u = HALF_STEP[dtype]
    tiny = 2.0 ** -25 * seen * vmax if dtype == arc.F16 else 0.0
    return u * np.abs(ref) + (1.01 * u + 2 * off + seen * 2.0 ** -23 + 2.0 ** -20) * mass + tiny + 2.0 ** -24


# -------------------------------------------------------------------- steps
class Step:
    """A step on the GPU: requests of `old` + `new` positions, pages in a random order (one pool of
    `spare` more), every value that no request may see NaN.  pages_per_row: table row length."""

    def __init__(self, old, new, page, kv_heads, hpk, dim, dtype, seed, rows=None, spare=3, stride_pad=0, ld_pad=0,
                 max_pages=None, max_new=None, sharp=1.0):
        rng = np.random.default_rng(seed)
        self.old, self.new, self.page, self.kv_heads, self.hpk, self.dim, self.dtype = old, new, page, kv_heads, hpk, dim, dtype
        self.heads = kv_heads * hpk
        lens = [o + n for o, n in zip(old, new)]
        need = [pages_of(n, page) for n in lens]
        self.num_pages = max(1, sum(need) + spare)
        order = rng.permutation(self.num_pages).astype(np.uint32)
        self.max_pages = max_pages or max(1, max(need, default=1))
        self.tables = rng.integers(0, 2 ** 32, (max(1, len(old)), self.max_pages), dtype=np.uint32)  # unused entries: anything
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at: at + n]
            at += n
        self.kvd = kv_heads * dim
        self.page_stride = page * self.kvd + stride_pad
        nan = 0x7E00 if dtype == arc.F16 else 0x7FC0
        self.k = np.full((self.num_pages, self.page_stride), nan, np.uint16)
        self.v = self.k.copy()
        self.K, self.V = [], []
        for b, n in enumerate(lens):
            K, V = (to_bits(rng.standard_normal((n, self.kvd)), dtype) for _ in range(2))
            for p in range(n):
                place = (p % page) * self.kvd
                self.k[self.tables[b, p // page], place: place + self.kvd] = K[p]
                self.v[self.tables[b, p // page], place: place + self.kvd] = V[p]
            self.K.append(from_bits(K, dtype).reshape(n, kv_heads, dim))
            self.V.append(from_bits(V, dtype).reshape(n, kv_heads, dim))
        self.used = sum(new)
        self.rows = self.used if rows is None else rows
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.lens = np.array(lens, np.uint32)
        self.width = self.heads * dim
        self.ldq, self.ldo = self.width + ld_pad, self.width + 2 * ld_pad
        self.q = to_bits(rng.standard_normal((self.rows, self.ldq)) * sharp, dtype)
        self.max_new = max(new, default=0) if max_new is None else max_new

    def upload(self):
        D = arc.DeviceBuffer.from_array
        self.dk, self.dv = D(self.k), D(self.v)
        self.pages = arc.KvPages(self.dk, self.dv, self.num_pages, self.page, self.kv_heads, self.dim, self.dtype,
                                 self.page_stride)
        self.dtables, self.dlens, self.dstarts = D(self.tables), D(self.lens), D(self.starts)
        self.batch = arc.PagedBatch(len(self.old), self.rows, self.max_pages, self.max_new, self.dtables, self.dlens,
                                    self.dstarts)
        self.dq = D(self.q)
        return self

    def attention(self, scale=0.0, window=0, sinks=0, workspace=None, stream=None):
        """Runs the step's attention; the output's bits [rows, ldo], 0xABCD where nothing was written."""
        out = arc.DeviceBuffer.from_array(np.full((max(1, self.rows), self.ldo), 0xABCD, np.uint16))
        ws = workspace or arc.DeviceBuffer(arc.paged_attention_workspace_bytes(self.pages, self.batch, self.hpk))
        if workspace is None:  # any contents will do
            ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
        arc.paged_attention(self.pages, self.batch, self.dq, self.ldq, self.hpk, out, self.ldo, ws, scale=scale,
                            window=window, sinks=sinks, stream=stream)
        if stream is not None:
            stream.synchronize()
        return out.download(np.uint16).reshape(-1, self.ldo)[: self.rows]

    def check(self, bits, scale=0.0, window=0, sinks=0, rows=None, dropped=None):
        """Every row (or the given ones) against float64; what no row covers is untouched.  dropped[b]:
        positions of request b whose page is not one of the pool.  Returns the largest share of the bound."""
        s = scale or self.dim ** -0.5
        worst = 0.0
        assert np.all(bits[self.used:] == 0xABCD), "rows behind the last request"
        assert np.all(bits[:, self.width:] == 0xABCD), "columns behind the heads"
        for b, (o, n) in enumerate(zip(self.old, self.new)):
            vmax = np.abs(self.V[b]).max() if len(self.V[b]) else 0.0
            for i in range(n):
                row = int(self.starts[b]) + i
                if rows is not None and row not in rows:
                    continue
                q = from_bits(self.q[row, : self.width], self.dtype).reshape(self.heads, self.dim)
                ref, mass, off, seen = attend(q, self.K[b], self.V[b], o + i, s, window, sinks,
                                              None if dropped is None else dropped[b])
                got = from_bits(bits[row, : self.width], self.dtype).reshape(self.heads, self.dim)
                tol = attention_bound(ref, mass, off, seen, vmax, self.dtype)
                assert np.all(np.isfinite(got)), (b, i)
                err = np.abs(got - ref)
                share = float((err / tol).max())
                assert share <= 1.0, (b, i, o + i, share, float(err.max()))
                worst = max(worst, share)
        return worst
