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
for n in ("kernels", "launches", "attributes", "workgroups", "most_threads"):
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


GEMM = """
def gemm(M, N, K):
    ld = -(-K // 16) * 16
    return lib.fbhip_gemm_i8(P(4096), L(ld), P(4096), P(4096), L(ld), P(4096), None, I(0), P(4096), L(N), I(0), I(M), I(N), I(K), P(4096), None)
SIZES = [(3600, 3500, 130), (2500, 1301, 333), (1500, 1500, 200), (300, 200, 200)]          # tiles of 256, 128 and 64 (two and four steps deep)
"""


def test_every_device_gets_the_tiles_shared_memory(run):
    """the limit is a device's own: a process that goes on to a second device has to raise it there too, once"""
    out = run(GEMM + """
for device in (0, 1, 0, 7, 1):
    hip.stand_in_device(device)
    for size in SIZES:
        rc = gemm(*size)
        assert rc == 0, (device, size, rc, lib.fbhip_last_error(None))
print(hip.stand_in_attributes(), hip.stand_in_launches())
""")
    assert out.split() == ["12", "20"], out          # four kernels on three devices; no K of these is split


def test_a_refused_limit_is_asked_for_again(run):
    run(GEMM + """
for size in SIZES:
    hip.stand_in_refuse_attribute(1)
    assert gemm(*size) != 0 and lib.fbhip_last_error(None)
    hip.stand_in_refuse_attribute(0)
    assert gemm(*size) == 0
""")


def test_the_sizes_of_the_gpu_tests_reach_every_kernel_of_the_product(run):
    """as many kernels as a sweep over all sizes launches"""
    from tests.test_gemm_i8_variants_gpu import SIZES
    out = run(GEMM + f"""
for size in {SIZES}:
    assert gemm(*size) == 0, size
print(hip.stand_in_kernels())
hip.stand_in_reset_kernels()
steps = [1, 2, 16, 17, 32, 33, 64, 65, 100, 200, 400, 800, 1600, 2400, 3200, 5000, 8191, 8192, 8193, 20000]
for M in steps:
    for N in steps:
        for K in (1, 100, 128, 129, 1000, 4096, 5000, 16384, 16385, 131071):
            assert gemm(M, N, K) == 0, (M, N, K)
print(hip.stand_in_kernels())
""")
    here, everywhere = map(int, out.split())
    assert here == everywhere == 10, out          # five strips, four tiles, the sum over slices of K


def test_no_launch_has_more_threads_than_one_may(run):
    """2^32 of them: 67 million short rows to quantise, a hundred million channels, long rows by the million"""
    run(GEMM + """
def quantise(rows, K, kind):
    Kp = -(-K // 128) * 128
    return lib.fbhip_quantize_rows(P(4096), L(K), I(kind), P(4096), L(Kp), P(4096), I(rows), I(K), I(Kp), None)
def linear(M, N, K):
    ld = -(-K // 16) * 16
    return lib.fbhip_linear_i8(P(4096), L(K), I(0), P(4096), L(ld), P(4096), None, I(0), P(4096), L(N), I(0), I(M), I(N), I(K), P(4096), None)
for rows, K in ((1 << 26, 3), ((1 << 26) + 5, 3), ((1 << 31) - 1, 3), (1 << 24, 1100), (1 << 24, 30000), ((1 << 23) + 1, 700)):
    for kind in (0, 1):
        assert quantise(rows, K, kind) == 0, (rows, K, kind, lib.fbhip_last_error(None))
for N in ((1 << 26) + 1, 1 << 27, 1 << 28, 1 << 30):
    for M in (1, 16, 40, 64, 200):
        assert gemm(M, N, 16) == 0, (M, N)
        assert linear(M, N, 16) == 0, (M, N)
assert hip.stand_in_most_threads() < 1 << 32
for M, N in ((1, (1 << 30) + 1), ((1 << 31) - 1, 1), (1, (1 << 31) - 1)):          # refused, not wrapped
    assert gemm(M, N, 16) == -1 and linear(M, N, 16) == -1 and b"too large" in lib.fbhip_last_error(None)
""")


def test_rows_of_every_piece_are_quantised_once(run):
    """the workgroups of all launches are those that the rows need"""
    out = run("""
for rows in (1, 4, 5, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 26) + 5):
    before = hip.stand_in_workgroups()
    assert lib.fbhip_quantize_rows(P(4096), L(3), I(0), P(4096), L(128), P(4096), I(rows), I(3), I(128), None) == 0
    print(hip.stand_in_workgroups() - before - -(-rows // 4))
""")
    assert out.split() == ["0"] * 7, out
