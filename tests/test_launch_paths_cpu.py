"""The library's host code on a machine without a GPU: tests/c_consumer/stand_in_runtime.cpp answers for the HIP runtime in a process of its own."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HEAD = """
import ctypes as C, sys
hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
lib = C.CDLL(sys.argv[2])
for n in ("launches", "attributes", "workgroups", "most_threads"):
    getattr(hip, "stand_in_" + n).restype = C.c_int64
lib.fbhip_last_error.restype = C.c_char_p
P, L, I = C.c_void_p, C.c_int64, C.c_int32
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    so = tmp_path_factory.mktemp("hip") / "libstand_in.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-O1", "-o", str(so), str(ROOT / "tests" / "c_consumer" / "stand_in_runtime.cpp")], check=True)
    lib = ROOT / "controllable_agent_amd" / "libfbhip.so"
    if not lib.exists():
        import __graft_entry__
        __graft_entry__.build_lib()

    def go(text):
        env = dict(os.environ, LD_LIBRARY_PATH="/opt/rocm/lib:" + os.environ.get("LD_LIBRARY_PATH", ""))
        env.pop("FBHIP_BRANCHED_GRAPHS", None)
        out = subprocess.run([sys.executable, "-c", HEAD + text, str(so), str(lib)], capture_output=True, text=True, timeout=120, env=env)
        assert out.returncode == 0, out.stdout + out.stderr
        return out.stdout
    return go


@pytest.mark.parametrize("version,allowed", [(70051831, 1), (70000000, 1), (60443484, 0), (70151831, 0), (70253211, 0), (80000000, 0)])
def test_branched_graphs_run_on_the_runtime_that_they_were_run_on(run, version, allowed):
    out = run(f"""
hip.stand_in_version({version})
why = C.c_char_p()
print(lib.fbhip_branched_graphs(C.byref(why)), why.value.decode())
""")
    got, why = out.strip().split(" ", 1)
    assert int(got) == allowed and why.startswith("allowed: HIP 7.0" if allowed else "refused: unverified"), out
