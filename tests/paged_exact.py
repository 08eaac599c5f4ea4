"""Paged attention whose scores are known exactly, so that only the roundings of weights, sums and
outputs are left: steps with given q, K and V, their rows in float64, and how far a row may be off."""
import numpy as np

import arcllm_amd as arc
import paged_lib as pl

LOG2E = 1.4426950408889634


class GivenStep(pl.Step):
    """A step with its q, K and V replaced: give() before upload()."""

    def give(self, b, K=None, V=None):
        """Request b's rows, [positions, kv_heads, dim], every value one of the type's."""
        pos = np.arange(int(self.lens[b]))
        page, place = self.tables[b, pos // self.page], pos % self.page
        for rows, pool, held in ((K, self.k, self.K), (V, self.v, self.V)):
            if rows is None:
                continue
            bits = pl.to_bits(rows, self.dtype).reshape(len(pos), self.kvd)
            assert np.array_equal(pl.from_bits(bits, self.dtype).reshape(rows.shape), rows)
            pool[:, : self.page * self.kvd].reshape(self.num_pages, self.page, self.kvd)[page, place] = bits
            held[b] = np.asarray(rows, np.float64)

    def give_q(self, q):
        """[rows, heads, dim] or what broadcasts to that."""
        q = np.ascontiguousarray(np.broadcast_to(q, (self.rows, self.heads, self.dim)), np.float64)
        bits = pl.to_bits(q.reshape(self.rows, self.width), self.dtype)
        assert np.array_equal(pl.from_bits(bits, self.dtype).reshape(q.shape), q)
        self.q[:, : self.width] = bits

    def rows_checked(self, rows):
        for b, (old, new) in enumerate(zip(self.old, self.new)):
            for i in range(new):
                if rows is None or int(self.starts[b]) + i in rows:
                    yield b, int(self.starts[b]) + i, old + i

    def check_exact(self, bits, scale, depth, window=0, sinks=0, rows=None):
        """Rows against float64, for scores that fp32 holds exactly whatever the order of their sum.  depth:
        the most additions in a row that a sum goes through.  Returns the largest share of the bound."""
        worst = 0.0
        for b, row, pos in self.rows_checked(rows):
            see = pl.visible(pos, int(self.lens[b]), window, sinks)
            q = pl.from_bits(self.q[row, : self.width], self.dtype).reshape(self.kv_heads, self.hpk, self.dim)
            got = pl.from_bits(bits[row, : self.width], self.dtype).reshape(q.shape)
            for g in range(self.kv_heads):
                ref, tol = exact_row(q[g], self.K[b][see, g], self.V[b][see, g], scale, depth, self.dtype)
                assert np.all(np.isfinite(got[g])), (b, pos, g)
                share = np.abs(got[g] - ref) / tol
                assert share.max() <= 1.0, (b, pos, g, float(share.max()), float(np.abs(got[g] - ref).max()))
                worst = max(worst, float(share.max()))
        return worst


LIFT = {arc.F16: 7, arc.BF16: 0}  # weights of the largest score are at least 2 to this


def exact_row(q, k, v, scale, depth, dtype):
    """q [heads, D], k and v [n, D]: the outputs and their bounds, [heads, D].
    A weight is 2^x, x = (score - largest) scale log2 e, off by
      * 2^-22 (|x| + 8) relative: the rounded constant scale log2 e, the difference, its product and the lift each
        2^-24 of at most |x| + 7, times ln 2; and exp2 itself 2^-23;
      * its rounding to the type, half a step: u relative, or half of fp16's smallest step, 2^-25, below its
        normal range, where the largest weight is 2^LIFT or more;
    the sum of weights takes them unrounded, so the first enters twice, the second once; both sums add up in fp32,
    2^-24 for each addition in a row; then the quotient 2^-22 and the output's rounding."""
    s = q @ k.T  # exact
    x = (s - s.max(1, keepdims=True)) * (scale * LOG2E)
    w = np.exp2(np.maximum(x, -2000.0))
    total = w.sum(1, keepdims=True)
    ref, size = w @ v / total, np.abs(v)
    u = pl.HALF_STEP[dtype]
    step = np.maximum(u * w, 2.0 ** (-25 - LIFT[dtype]) if dtype == arc.F16 else 0.0)
    rel = w * (np.minimum(-x, 2000.0) + 8) * 2.0 ** -22
    mass = w @ size / total
    tol = (step + rel) @ size / total + np.abs(ref) * rel.sum(1, keepdims=True) / total
    return ref, tol + (2 * depth * 2.0 ** -24 + 2.0 ** -22) * mass + 1.01 * u * np.abs(ref) + 2.0 ** -24


# ------------------------------------------------------------ position codes
def coded_rows(n, kv_heads, dim, course):
    """K and V, [n, kv_heads, dim], for q = 1: V is 1 in one dim, that of a block of 32 positions in even kv heads, of the
    position itself in odd ones, so that an output is the weight of the positions with its code and one that is
    left out or taken twice shows.  Scores are whole numbers: equal, or 0 .. 7 along the context, rising or falling."""
    pos = np.arange(n)
    level = {"equal": pos * 0, "rising": pos * 8 // n, "falling": 7 - pos * 8 // n}[course]
    K, V = np.zeros((n, kv_heads, dim)), np.zeros((n, kv_heads, dim))
    K[:, :, 0] = level[:, None]
    for g in range(kv_heads):
        V[pos, g, (pos if g % 2 else pos // 32) % dim] = 1.0
    return K, V


def coded_step(old, new, kv_heads, hpk, dim, dtype, course, page=16):
    s = GivenStep(old, new, page, kv_heads, hpk, dim, dtype, 1)
    s.give_q(1.0)
    for b, n in enumerate(s.lens):
        s.give(b, *coded_rows(int(n), kv_heads, dim, course))
    return s


# long contexts that are cut into many parts: old, new, kv_heads, hpk, dim, window, sinks
CODED = [([131070], [1], 1, 2, 64, 0, 0), ([40000, 12345, 70], [1, 1, 1], 2, 4, 128, 0, 0), ([20000, 333], [1, 3], 2, 8, 64, 0, 0),
         ([50000, 9000], [1, 5], 2, 4, 128, 7000, 100), ([12000], [200], 2, 4, 128, 0, 0), ([9000, 2000], [70, 130], 2, 2, 64, 0, 0),
         ([15000], [300], 2, 2, 64, 3000, 70), ([0, 4000], [600, 1], 2, 4, 128, 0, 0)]
