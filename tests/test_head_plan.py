"""What the head's loss refuses and what its plans hold (anni_amd/csrc/head_plan.h), on the host: the checks
end before any device is looked for, so a refusal can be told from a missing device, and the
invented addresses of the jobs never reach a launch."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("head_plan") / "head_plan_test")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined",
                           "-fno-sanitize-recover=undefined", "-I", os.path.join(ROOT, "include"),
                           "-I", os.path.join(ROOT, "anni_amd", "csrc"),
                           os.path.join(ROOT, "tests", "c", "head_plan_test.cpp"), "-o", exe])
    return exe


def test_jobs_that_are_refused_and_taken(program):
    """A job with gradients and the size functions' -1 as their type among the refused: its plan has no part
    for gradients, and the launches divide by one."""
    r = subprocess.run([program], stdout=subprocess.PIPE, timeout=120)
    out = r.stdout.decode()
    assert r.returncode == 0 and out.startswith("ok refused "), out


def plans(program, sizes):
    """Each size's shapes, as (name, number) pairs of what the program prints."""
    out = subprocess.check_output([program] + [str(v) for s in sizes for v in s], timeout=120).decode().splitlines()
    lines = [dict(zip(ln.split()[::2], map(int, ln.split()[1::2]))) for ln in out]
    assert len(lines) == len(sizes)
    return lines


def test_the_sizes_compared_with_the_model_reach_every_kernel(program):
    """The lists of test_gpu_head_shapes.py against the plan's rules: whatever the rules become, a kernel that no
    listed size is made of fails here."""
    from test_gpu_head_shapes import GRADIENTS, LOSSES
    seen = set()
    for (_r, _d, _v, ty, _p), p in zip(GRADIENTS, plans(program, [g[:4] for g in GRADIENTS])):
        several = p["pieces"] > 1
        for kept in ([1] if p["always"] else [0, 1] if p["keeps"] else [0]):
            seen.add(("logits", p["logits"], ty, kept))
        seen |= {("dx", p["dx"], ty), ("dx slices", p["slices_dx"], ty), ("dw", p["dw"], p["slices_dw"], ty),
                 ("pieces", several, p["dw"], p["slices_dw"], ty), ("copied", p["copied"], ty)}
    want = {("logits", 64, ty, 1) for ty in (0, 1)}
    want |= {("logits", t, ty, k) for t in (128, 256) for ty in (0, 1) for k in (0, 1)}
    want |= {("dx", k, ty) for k in (0, 1, 2) for ty in (0, 1)}
    want |= {(name, k, ty) for name in ("dx slices", "copied") for k in (0, 1) for ty in (0, 1)}
    shapes = [(128, 0), (128, 1), (256, 0)]
    want |= {("dw",) + s + (ty,) for s in shapes for ty in (0, 1)}
    want |= {("pieces", True) + s + (ty,) for s in [(128, 1), (256, 0)] for ty in (0, 1)}
    assert not want - seen, want - seen
    losses = plans(program, [(r, d, v, -1) for r, d, v, _b in LOSSES])
    assert {(p["logits"], p["copied"]) for p in losses} >= {(64, 0), (128, 0), (128, 1), (256, 0), (256, 1)}
    assert not any(p["keeps"] for p in losses)
