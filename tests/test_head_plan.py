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
