"""How attention_shared cuts its work, on the CPU (tests/native/check_split_host.cu)."""
import glob
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cut_and_join(tmp_path):
    from metalqwen3_b200.build import CSRC, build_library
    build_library()
    objs = [o for o in glob.glob(os.path.join(CSRC, "_build", "*.o")) if os.path.basename(o) != "k_shared.o"]
    exe = str(tmp_path / "check_split_host")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--fmad=false", "-Xptxas", "-O0", "-I", CSRC,
                    "-I", os.path.join(ROOT, "include"), "-o", exe,
                    os.path.join(ROOT, "tests", "native", "check_split_host.cu")] + objs, check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
