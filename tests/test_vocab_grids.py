"""Every launch of cavs_vocab_xent* fits a grid, whose threads along a dimension are fewer than 2^32.  Host only: the calls run up to their launches."""
import os
import subprocess

from cavs_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_grids_over_the_range_of_sizes(tmp_path):
    exe = str(tmp_path / "vocab_grids")
    lib = os.path.dirname(build.HIP_SO)
    cmd = [build.HIPCC, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-I", os.path.join(build.ROOT, "include"), "-I", build.CSRC,
           os.path.join(HERE, "native", "vocab_grids.cc"), "-o", exe, "-L", lib, "-lcavs_hip", "-Wl,-rpath," + lib,
           "-Wl,--unresolved-symbols=ignore-in-object-files"]  # (the kernels' code, which nothing launches)
    subprocess.run(cmd, check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.endswith("0 grids too large\n"), r.stdout[-2000:] + r.stderr[-500:]
    assert int(r.stdout.split()[-6]) > 1000, r.stdout[-200:]
