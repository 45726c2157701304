"""When an orthogonalised update makes do with two parts: bf16 results alone, and steps that let a rounding grow to no more than 2^9 of itself.  Host only."""
import os
import subprocess

import pytest

from cavs_amd import build, hip

HERE = os.path.dirname(os.path.abspath(__file__))
NS, CUBIC, QUINTIC = (3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    exe, lib = str(tmp_path_factory.mktemp("growth") / "ortho_growth"), os.path.dirname(build.HIP_SO)
    cmd = [build.HIPCC, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(build.ROOT, "include"), "-I", build.CSRC,
           os.path.join(HERE, "native", "ortho_growth.cc"), "-o", exe, "-L", lib, "-lcavs_hip", "-Wl,-rpath," + lib,
           "-Wl,--unresolved-symbols=ignore-in-object-files"]  # (the kernels' code, which nothing launches)
    subprocess.run(cmd, check=True, capture_output=True)

    def ask(type_, weights, *cases):
        args = [str(type_), str(int(weights))] + [str(v) for steps, ns in cases for v in (steps, *ns)]
        return [int(v) for v in subprocess.run([exe] + args, check=True, capture_output=True, text=True, timeout=60).stdout.split()]

    return ask


def test_where_two_parts_do(parts):
    # a^steps: 485 and 1670; 438 and 657; 286 and 537
    cases = [(1, NS), (5, NS), (6, NS), (64, NS), (15, CUBIC), (16, CUBIC), (30, CUBIC), (9, QUINTIC), (10, QUINTIC)]
    assert parts(hip.BF16, False, *cases) == [2, 2, 3, 3, 2, 3, 3, 2, 3]
    assert parts(hip.BF16, True, *cases) == [3] * len(cases)
    assert parts(hip.F32, False, *cases) == [3] * len(cases)


def test_coefficients_whose_steps_leave_a_floats_range(parts):
    """Wherever among the singular values that is, also where a slope behind it would be small again"""
    inf, nan = float("inf"), float("nan")
    assert parts(hip.BF16, False, (64, (0.1, 0.0, 30.0)), (64, (0.0, 0.0, 1e30)), (3, (nan, 0.0, 0.0)), (3, (0.5, nan, 0.0)), (3, (0.5, inf, -inf)),
                 (8, (1.0, -30.0, 0.0)), (64, (-0.5, 20.0, -20.0))) == [3] * 7
