"""The paged-cache operators' index arithmetic and refusals, on the CPU (tests/native/check_paged_host.cu)."""
import glob
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_indices_and_refusals(tmp_path):
    from metalqwen3_b200.build import CSRC, build_library
    build_library()
    objs = [o for o in glob.glob(os.path.join(CSRC, "_build", "*.o")) if os.path.basename(o) != "q3cu_api.o"]
    exe = str(tmp_path / "check_paged_host")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--fmad=false", "-I", CSRC,
                    "-I", os.path.join(ROOT, "include"), "-o", exe,
                    os.path.join(ROOT, "tests", "native", "check_paged_host.cu")] + objs, check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_bindings_match_the_header():
    """The ctypes structures have the C layout."""
    import ctypes as C
    from metalqwen3_b200.q3cu import _KVBatch, _KVCache
    assert C.sizeof(_KVCache) == 48 and _KVCache.dtype.offset == 40
    assert C.sizeof(_KVBatch) == 32 and _KVBatch.max_pages.offset == 28
