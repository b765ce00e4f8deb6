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


SERVER = r'''
#include "CudaContext.h"
// A layer of a serving step through the C++ context: append a batch's rows, attend from prompts or from new tokens.
void layer(CudaContext &ctx, const q3cu_kv_cache &cache, const q3cu_kv_batch &batch, int64_t rows, const float *qkv,
           const float *qn, const float *kn, void *q, void *work, size_t work_bytes, void *out, bool prompts,
           q3cu_stream stream) {
    const int heads = 32, n_kv = 8;
    const int64_t stride = (heads + 2 * n_kv) * 128;
    ctx.kvAppend(cache, batch, rows, qkv, qkv + heads * 128, qkv + (heads + n_kv) * 128, Q3CU_F32, stride, stride, heads, qn,
                 kn, q, Q3CU_BF16, stream);
    if (prompts) ctx.attentionPrompt(cache, batch, rows, q, Q3CU_BF16, heads * 128, heads, out, stream);
    else ctx.attentionPaged(cache, batch, q, Q3CU_BF16, heads * 128, heads, work, work_bytes, out, stream);
}
int main() {
    CudaContext ctx(0);
    return ctx.isInitialized() ? int(ctx.attentionPagedWorkspace(32, 8) == 0) : 0;
}
'''


def test_cpp_boundary_compiles_and_links(tmp_path):
    from metalqwen3_b200.build import build_library
    lib = os.path.dirname(build_library())
    src = tmp_path / "server.cpp"
    src.write_text(SERVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(tmp_path / "server"), "-L", lib, "-lq3cu", f"-Wl,-rpath,{lib}"], check=True)
    assert subprocess.run([str(tmp_path / "server")], timeout=60).returncode == 0
