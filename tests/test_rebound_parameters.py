"""The optimizer moves the tensors a parameter is bound to when it runs.  Host only: the host runtime over a stand-in for the device."""
import os
import re
import subprocess

from cavs_amd import build, hip

HERE = os.path.dirname(os.path.abspath(__file__))


def test_orthogonalised_updates_follow_bind_param(tmp_path):
    native = [os.path.join(HERE, "native", f) for f in ("rebind_check.cc", "device_standin.cc")]
    own = set(re.findall(r"\b(cavs_[a-z0-9_]+)\(", "".join(open(f).read() for f in native)))
    rest = tmp_path / "rest.c"  # every other entry point of the device: nothing is done
    rest.write_text("".join(f"int {n}() {{ return 0; }}\n" for n in sorted(set(hip._SIGS) - own)))
    subprocess.run(["gcc", "-fPIC", "-c", str(rest), "-o", str(tmp_path / "rest.o")], check=True, capture_output=True)
    exe, lib = str(tmp_path / "check"), os.path.dirname(build.HOST_SO)
    subprocess.run([build.CXX] + build.CXX_FLAGS + native + [str(tmp_path / "rest.o"), "-rdynamic", "-o", exe, "-L", lib, "-lcavs_host", "-lcavs_hip",
                                                             "-Wl,-rpath," + lib], check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "0 wrong\n", r.stdout + r.stderr
