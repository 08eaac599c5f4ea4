"""The plan of the 8-bit products: which kernel takes the products that the GPU tests of every form run, that those
tests leave no form out, and that a workspace of up to so many rows holds what each of them needs."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

import arcllm_amd as arc
import fp8_forms as ff

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("fp8_plan") / "fp8_plan"
    subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT}/arcllm_amd/csrc",
                    str(ROOT / "tests" / "cpp" / "fp8_plan.cpp"), "-o", str(exe)], check=True)

    def ask(products):
        lines = "\n".join(" ".join(map(str, p[:5])) for p in products)
        out = subprocess.run([str(exe)], input=lines, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(products)
        return [(form, *map(int, rest)) for form, *rest in map(str.split, out)]

    return ask


def turns(form, parts):
    """How often the workgroups of k_fp8_deep go on to a further tile."""
    wgs = {"deep128": 512, "deep256": 256}.get(form)
    return (parts - 1) // wgs if wgs and parts > wgs else None


def test_forms_of_the_gpu_tests(plan):
    for case, (form, mtiles, ntiles, splits, *_) in zip(ff.ALL, plan(ff.ALL)):
        assert case[5:] == (form, splits, turns(form, mtiles * ntiles * splits)), case


def products(rng, n):
    for _ in range(n):
        m, cols, k = int(2 ** rng.uniform(0, 12.5)), int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 10.5))
        k = 128 * max(1, k // 8) if rng.random() < 0.6 else 16 * k
        yield m, cols, k, int(rng.random() < 0.5), int(rng.random() < 0.5)


def test_no_form_is_left_out(plan):
    """Each form, gated and not, by type of y, by number of parts where there are several, and with columns that end inside a block."""
    some = list(products(random.Random(3), 60000))
    kind = lambda p, form, splits: (form, p[3], p[4], splits, p[2] % 128 != 0 if form.startswith("rows") else None)  # noqa: E731
    tested = {kind(p, p[5], p[6]) for p in ff.ALL}
    whole = {t[:4] for t in tested}
    for p, (form, _, _, splits, *_) in zip(some, plan(some)):
        assert kind(p, form, splits)[:4] in whole, p
        if splits == 1:
            assert kind(p, form, splits) in tested, p


def test_workspace_holds_what_any_plan_needs(plan):
    rng = random.Random(4)
    for _ in range(60):
        _, n, k, gated, fast = next(products(rng, 1))
        most = sorted(int(2 ** rng.uniform(0, 15)) for _ in range(3))
        asked = [(m, n, k, gated, fast) for m in (*range(1, most[-1], max(1, most[-1] // 300)), *most)]
        for top in most:
            size = arc.fp8_gemm_workspace_bytes(n, k, top, bool(gated))
            assert all(a[4] <= size for p, a in zip(asked, plan(asked)) if p[0] <= top), (n, k, gated, top)
