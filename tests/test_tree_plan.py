"""The plan of pa_decode_tree and the records that a context holds for it, worked out by the library's own source without a GPU (tree_plan.cu)."""
import json
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    from pooled_b200 import build
    try:
        nvcc = build.nvcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = str(tmp_path_factory.mktemp("plan") / "tree_plan")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-w", os.path.join(ROOT, "tests", "tree_plan.cu"), "-o", out],
                   check=True, capture_output=True)

    def run(nH, nKV, hd, f16, cols, sizes=(), records=0):
        """(the context's records, the launches)"""
        text = subprocess.run([out, *map(str, (nH, nKV, hd, int(f16), cols, records)), *[f"{b}.{n}" for b, n in sizes]], check=True, capture_output=True, text=True).stdout
        held, *launches = map(json.loads, text.splitlines())
        return held, launches
    return run


@pytest.mark.parametrize("nH,cols,prefill,tree", [
    (1, 1, 16384, 18944), (16, 1, 16384, 18944), (16, 8, 16384, 18944), (24, 8, 16384, 26112), (16, 16, 16384, 32768), (16, 128, 16384, 32768), (24, 400, 32768, 38400),
    (16, 960, 32768, 61440), (16, 8192, 32768, 65536), (128, 8, 16384, 32768)])
def test_records_of_a_context(plan, nH, cols, prefill, tree):
    held, _ = plan(nH, 1, 64, True, cols)
    assert held == {"part": 16384, "prefill": prefill, "tree": tree}


def test_contexts_of_few_columns_plan_their_trees_as_if_they_held_more_records(plan):
    # trees of no more tokens than the context has columns, behind up to 34000 rows
    r = random.Random(1)
    shapes = [(16, 8, 128), (16, 2, 256), (24, 4, 256), (4, 4, 64), (10, 2, 128), (64, 1, 64), (1, 1, 64), (8, 1, 256), (32, 8, 128), (2, 2, 256)]
    fewer = 0
    for _ in range(400):
        nH, nKV, hd = r.choice(shapes)
        sizes = [(int(2 ** r.uniform(0, 15.05)), int(2 ** r.uniform(0, 3.5))) for _ in range(r.choice([1, 1, 2, 3]))]
        cols = max(r.choice([1, 8]), sum(n for _, n in sizes))
        f16 = r.random() < 0.5
        held, launches = plan(nH, nKV, hd, f16, cols, sizes)
        if held["tree"] < 32768:
            fewer += 1
            assert plan(nH, nKV, hd, f16, cols, sizes, records=32768)[1] == launches, (nH, nKV, hd, f16, sizes)
    assert fewer > 100


def test_the_long_runs_of_the_gpu_tests_are_reached(plan):
    # wide and narrow row tiles, units of several runs (added up in one record, or a record each) and of one, at every head_dim that tests name
    from tests.test_gpu_tree_runs import CASES
    reached = set()
    for name, (nH, nKV, hd, f16, cols, sizes, wide, several, run) in CASES.items():
        _, launches = plan(nH, nKV, hd, f16, cols, sizes)
        kernels = [(bool(p["wide"]), p["fold"] > 1 or (bool(p["wide"]) and p["tiles"] > p["run"])) for p in launches]       # (WIDE, FOLD)
        assert kernels[0] == (wide, several) and max(p["run"] for p in launches) == run, (name, launches)
        reached.update((hd, *k) for k in kernels)
        reached.update((hd, "added up" if p["fold"] > 1 else "one by one") for p in launches if p["wide"])
    assert {(hd, True, True) for hd in (256, 128, 64)} <= reached and {(hd, False, True) for hd in (256, 128, 64)} <= reached
    assert {(256, "added up"), (128, "added up"), (64, "added up"), (128, "one by one")} <= reached
