"""The split of a block end's gradient over teams, and its workspace, on the CPU: flagcx_amd/csrc/host_residual.cpp compiled
with launchers that note what they are given (tests/residual_host_harness/harness.cpp)."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = [os.path.join(ROOT, "tests", "residual_host_harness", "harness.cpp"),
           os.path.join(ROOT, "flagcx_amd", "csrc", "host_residual.cpp")]


@pytest.fixture(scope="module")
def sizes(tmp_path_factory):
    gxx = shutil.which("g++")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    if not gxx or not os.path.exists(os.path.join(rocm, "include", "hip", "hip_runtime.h")):
        pytest.skip("no g++ or no HIP headers")
    exe = str(tmp_path_factory.mktemp("residual_harness") / "harness")
    r = subprocess.run([gxx, "-O1", "-std=c++17", "-w", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(rocm, "include")] +
                       SOURCES + ["-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]

    def run(cases):
        text = "".join("%d %d %d %d\n" % c for c in cases)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr[-2000:]
        got = [int(x) for x in out.stdout.split()]
        assert len(got) == len(cases)
        return got
    return run


GROUPS = (0, 1, 2, 3, 7, 20, 55, 100, 300, 1000, 2048, 5000, 1 << 40)


@pytest.mark.parametrize("dim", [1, 64, 512, 520, 1024, 2047, 4096, 6144, 8192, 8200, 16384])
def test_workspace_of_the_longest_batch_serves_shorter_ones(sizes, dim):
    """Every split's rows are each one team's and its partial rows lie in the workspace (the harness looks); the size does
    not fall from one batch to a longer one."""
    rows = sorted(set(list(range(0, 600)) + list(range(600, 4500, 13)) + [3585, 2234, 8191, 8192, 8193, 20000, 32768, 40000]))
    for gate, groups in [(0, 0), (0, 7)] + [(1, n) for n in GROUPS]:
        got = sizes([(n, dim, gate, groups) for n in rows])
        for a, b, n in zip(got, got[1:], rows[1:]):
            assert a <= b, (n, dim, gate, groups, a, b)
        # and stays near what the rows themselves take in fp32
        for b, n in zip(got, rows):
            assert b <= 12 * dim * n


def test_random_splits(sizes):
    rng = random.Random(5)
    cases = []
    for _ in range(6000):
        n = int(2 ** rng.uniform(0, 14))
        cases.append((n, rng.randint(1, 16384), 1, rng.choice((0, 1, rng.randint(2, 2 * n + 1), int(2 ** rng.uniform(1, 14))))))
    sizes(cases)
