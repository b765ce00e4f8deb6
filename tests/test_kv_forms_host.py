"""The paged cache's further forms without a GPU: arithmetic and refusals (tests/native/check_kv_forms_host.cu), and the
Python side with a library that only notes its arguments."""
import ctypes as C
import glob
import os
import subprocess

import pytest
import torch

from metalqwen3_b200 import q3cu
from test_paged_binding import Stream, Tensor, binding, cache_and_batch  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I8, I32, F32 = torch.int8, torch.int32, torch.float32


def test_arithmetic_and_refusals(tmp_path):
    from metalqwen3_b200.build import CSRC, build_library
    build_library()
    objs = [o for o in glob.glob(os.path.join(CSRC, "_build", "*.o")) if os.path.basename(o) != "q3cu_api.o"]
    exe = str(tmp_path / "check_kv_forms_host")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--fmad=false", "-I", CSRC,
                    "-I", os.path.join(ROOT, "include"), "-o", exe,
                    os.path.join(ROOT, "tests", "native", "check_kv_forms_host.cu")] + objs, check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


LAYOUT = r'''
#include "q3cu.h"
#include <cstddef>
#include <cstdio>
int main() {
    std::printf("%zu %zu %zu %zu %zu %zu %zu %zu\n", sizeof(q3cu_kv_cache_q8), offsetof(q3cu_kv_cache_q8, k_scale),
                offsetof(q3cu_kv_cache_q8, scale_stride), sizeof(q3cu_rope), offsetof(q3cu_rope, gain), offsetof(q3cu_rope, freq),
                sizeof(q3cu_kv_prefix), offsetof(q3cu_kv_prefix, n_groups));
}
'''


def test_structures_have_the_c_layout(tmp_path):
    src = tmp_path / "layout.cpp"
    src.write_text(LAYOUT)
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True).stdout.split()]
    q8, rope, prefix = q3cu._KVCacheQ8, q3cu._Rope, q3cu._KVPrefix
    assert got == [C.sizeof(q8), q8.k_scale.offset, q8.scale_stride.offset, C.sizeof(rope), rope.gain.offset, rope.freq.offset,
                   C.sizeof(prefix), prefix.n_groups.offset]


def quantised(device=0, **kw):
    codes = [Tensor((4, 2, 16, 128), I8, device) for _ in range(2)]
    scales = [Tensor((4, 2, 16, 2), F32, device) for _ in range(2)]
    return q3cu.KVCache(*codes, *scales)


def test_quantised_caches(binding):  # noqa: F811
    cache = quantised()
    assert cache.quantised and cache.c.dtype == 8 and cache.c.scale_stride == 64 and cache.c.page_stride == 4096
    codes, scale = Tensor((4, 2, 16, 128), I8), Tensor((4, 2, 16, 2), F32)
    for bad in (lambda: q3cu.KVCache(codes, codes), lambda: q3cu.KVCache(codes, codes, scale),
                lambda: q3cu.KVCache(codes, codes, scale, Tensor((4, 2, 16, 1), F32)),
                lambda: q3cu.KVCache(codes, codes, scale, Tensor((4, 2, 16, 2), F32, 1)),
                lambda: q3cu.KVCache(Tensor((4, 2, 16, 128)), Tensor((4, 2, 16, 128)), scale, scale)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        q3cu.KVCache(codes, codes, scale, Tensor((4, 2, 16, 2), torch.bfloat16))
    spread = Tensor((4, 2, 16, 2), F32)
    spread.t = torch.empty((4, 2, 16, 4))[..., ::2]
    with pytest.raises(ValueError):
        q3cu.KVCache(codes, codes, spread, spread)


@pytest.mark.parametrize("given", [False, True])
def test_calls_make_their_memory_on_their_stream(binding, given):  # noqa: F811
    binding.torch.__class__.bfloat16 = torch.bfloat16
    stream = Stream(9) if given else None
    on = stream or binding.main
    _, batch = cache_and_batch()
    cache, q, k = quantised(), Tensor((3, 4, 128)), Tensor((3, 2, 128))
    prefix = q3cu.KVPrefix(Tensor((2,), I32), Tensor((1,), I32))
    results = [binding.kv_append(cache, batch, q, k, k, stream=stream, rope=q3cu.Rope(dim=64)),
               *binding.kv_read(cache, batch, rows=3, stream=stream), binding.attention_paged(cache, batch, q, stream=stream),
               binding.attention_prompt(cache, batch, q, stream=stream)]
    results.append(binding.attention_shared(cache, batch, prefix, q, stream=stream, work=Tensor((1 << 20,), torch.uint8)))
    assert all(t.made_on is on for t in binding.torch.made) and all(t.dtype == torch.bfloat16 for t in results)
    if given:
        assert all(binding.main in t.used_on for t in results)
    names = [name for name, _ in binding.lib.calls if "workspace" not in name]
    assert names == ["q3cu_kv_append_rope", "q3cu_kv_read", "q3cu_attention_paged", "q3cu_attention_prompt",
                     "q3cu_attention_shared"]
    assert {args[-1] for name, args in binding.lib.calls if "workspace" not in name} == {on.cuda_stream}


def test_memory_elsewhere_is_refused(binding):  # noqa: F811
    _, batch = cache_and_batch()
    q = Tensor((3, 4, 128))
    near = q3cu.KVPrefix(Tensor((2,), I32), Tensor((1,), I32))
    far = q3cu.KVPrefix(Tensor((2,), I32, 1), Tensor((1,), I32, 1))
    for c, p in ((quantised(1), near), (quantised(), far)):
        with pytest.raises(ValueError, match="must be on the context's GPU"):
            binding.attention_shared(c, batch, p, q)
    with pytest.raises(ValueError, match="must be on the context's GPU"):
        binding.kv_read(quantised(1), batch, rows=3)
    with pytest.raises(ValueError, match="work must be contiguous"):
        binding.attention_shared(quantised(), batch, near, q, work=Tensor((64,), torch.uint8, 1))
    out = Tensor((3, 2, 128))
    for bad in (lambda: binding.kv_read(quantised(), batch), lambda: binding.kv_read(quantised(), batch, k_out=out),
                lambda: binding.kv_read(quantised(), batch, k_out=out, v_out=Tensor((3, 3, 128))),
                lambda: binding.kv_read(quantised(), batch, rows=4, k_out=out, v_out=out),
                lambda: binding.kv_read(quantised(), batch, k_out=out, v_out=Tensor((3, 2, 128), device=1))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        binding.kv_read(quantised(), batch, k_out=out, v_out=Tensor((3, 2, 128), F32))
    assert not [c for c in binding.lib.calls if "workspace" not in c[0]]


def test_rope_arguments():
    r = q3cu.Rope(theta=1e4, dim=4, interleaved=True, freq=[0.5, 0.25])
    assert r.c.layout == 1 and r.c.freq[1] == 0.25 and r.c.gain == 0.0
    assert q3cu.Rope(scaling="yarn", factor=4, original=4096).c.scaling == 2
    for bad in (dict(scaling="longest"), dict(gain=0.0), dict(gain=-1.0), dict(dim=8, freq=[1.0])):
        with pytest.raises(ValueError):
            q3cu.Rope(**bad)


SERVER = r'''
#include "CudaContext.h"
// A layer of a serving step over a Q8_0 cache through the C++ context.
void layer(CudaContext &ctx, const q3cu_kv_cache_q8 &cache, const q3cu_kv_batch &batch, const q3cu_kv_prefix &prefix, int64_t rows,
           const float *qkv, void *q, void *work, size_t bytes, void *out, q3cu_stream stream) {
    q3cu_rope rope{};
    rope.theta = 1e6f, rope.dim = 64, rope.layout = Q3CU_ROPE_PAIRS, rope.scaling = Q3CU_ROPE_LINEAR, rope.factor = 2.0f;
    ctx.kvAppend(cache.codes, batch, rows, qkv, qkv + 32 * 128, qkv + 40 * 128, Q3CU_F32, 48 * 128, 48 * 128, 32, nullptr, nullptr, q,
                 Q3CU_BF16, stream, rope);
    ctx.attentionShared(cache.codes, batch, prefix, q, Q3CU_BF16, 32 * 128, 32, work, bytes, out, stream);
    ctx.attentionPrompt(cache.codes, batch, rows, q, Q3CU_BF16, 32 * 128, 32, out, stream);
    ctx.kvRead(cache.codes, batch, rows, q, out, Q3CU_BF16, 8 * 128, stream);
}
int main() {
    CudaContext ctx(0);
    return ctx.isInitialized() ? int(ctx.attentionSharedWorkspace(64, 32, 8) == 0) : 0;
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
