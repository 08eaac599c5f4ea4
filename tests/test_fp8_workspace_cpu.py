"""The 8-bit products' workspace serves every call of up to its rows: its size never falls as rows grow."""
import random

import pytest

import arcllm_amd as arc


@pytest.mark.parametrize("n,k,gated", [(3584, 18944, False), (4608, 3584, False), (18944, 3584, True), (100, 4096, False), (8192, 8192, False),
                                       (31, 48, False), (40000, 65536, False), (1500, 8192, True), (700, 100000, False)])
def test_more_rows_need_no_less(n, k, gated):
    sizes = [arc.fp8_gemm_workspace_bytes(n, k, m, gated) for m in [*range(0, 1300), *range(1300, 30000, 61)]]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] >= 256


def test_any_weights():
    rng = random.Random(8)
    for _ in range(200):
        n, k, gated = int(2 ** rng.uniform(0, 17)), 16 * int(2 ** rng.uniform(0, 13)), rng.random() < 0.4
        rows = sorted(int(2 ** rng.uniform(0, 14)) for _ in range(20))
        sizes = [arc.fp8_gemm_workspace_bytes(n, k, m, gated) for m in rows]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), (n, k, gated, rows)


def test_the_largest_sizes_are_answered():
    assert arc.fp8_gemm_workspace_bytes(1 << 24, 1 << 22, 1 << 24) >= 256
    assert arc.fp8_gemm_workspace_bytes(1, 1 << 22, 1 << 24) >= arc.fp8_gemm_workspace_bytes(1, 1 << 22, 1 << 23)
