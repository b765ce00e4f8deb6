"""Appending with other rotations and into Q8_0 caches, and reading rows back, against the formulas in binary64.

Tolerances (u = 2^-24, H = 2^-8, half a step of bf16):
  * rotation: a tree sum of 128 squares, a root, a division and two products are within 16 u, sine and cosine within 4 u,
    the gain (itself rounded to binary32) adds 2 u: 28 u gain (|y| + |z|) of the pair's elements y, z before the turn; an
    element that is not turned: 16 u |y|, which the same bound covers with gain >= 1; a bf16 result H |o| more.
  * Q8_0 codes and scales are those that q3cu_quantize_q8 makes of the f32 rows: equal.
  * reading back is one product, and one rounding to bf16: equal to the same operations.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_paged import BF16, F32, H, U, Paged, offsets, queries

pytestmark = pytest.mark.gpu
I8 = torch.int8


class Quantised(Paged):
    """Sequences on shuffled pages of a Q8_0 pool: codes and scales of every slot that is not filled are `fill`ed."""

    def __init__(self, lens, n_kv, page, seed, spare=3, gap=0, code=77, scale=float("nan")):
        super().__init__(lens, n_kv, page, I8, seed, spare, gap, code)
        pitch = n_kv * page * 2 + gap // 8         # (a multiple of 4)
        self.scale_pool = [torch.full((self.n_pages, pitch), scale, device="cuda") for _ in range(2)]
        self.ks, self.vs = (p.as_strided((self.n_pages, n_kv, page, 2), (pitch, page * 2, 2, 1)) for p in self.scale_pool)

    def fill(self, seed, scale=1.0):
        """Random codes of every value and random scales at every position of every sequence."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        for s, n in enumerate(self.lens):
            if n > 0:
                page, slot = self.where(s, range(n))
                for t, c in ((self.k, self.ks), (self.v, self.vs)):
                    x = torch.randn((n, self.n_kv, 2, 64), generator=g, device="cuda") * scale
                    step = x.abs().amax(-1) / 127
                    c[page, :, slot] = step
                    code = torch.round(x / step.clamp_min(1e-30)[..., None]).clamp(-127, 127)
                    code[..., 0, 5] = -128              # a code that only wrapped groups have
                    t[page, :, slot] = code.flatten(-2).to(I8)
        return self

    def held(self, s, positions):
        """Keys and values [n][n_kv][128] as the products of code and scale in binary32."""
        page, slot = self.where(s, positions)
        return [t[page, :, slot].float() * c[page, :, slot].repeat_interleave(64, -1)
                for t, c in ((self.k, self.ks), (self.v, self.vs))]

    def rows(self, s):
        page, slot = self.where(s, range(max(self.lens[s], 0)))
        return tuple(t[page, :, slot].double() * c[page, :, slot].double().repeat_interleave(64, -1)
                     for t, c in ((self.k, self.ks), (self.v, self.vs)))

    def handles(self, row_off=None):
        from metalqwen3_b200.q3cu import KVBatch, KVCache
        off = None if row_off is None else torch.tensor(row_off, dtype=torch.int32, device="cuda")
        return KVCache(self.k, self.v, self.ks, self.vs), KVBatch(self.kv_len, self.table, off)


def yarn(theta, dim, factor, original, fast=32.0, slow=1.0):
    """YaRN's frequencies pair by pair."""
    def pair(turns):
        return dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))
    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
    out = []
    for j in range(dim // 2):
        f = theta ** (-2 * j / dim)
        share = min(max((j - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(f * (1 - share) + f / factor * share)
    return out


ROPES = {
    "halves": (dict(theta=1e4), [1e4 ** (-j / 64) for j in range(64)], 1.0),
    "pairs": (dict(theta=1e6, interleaved=True), [1e6 ** (-j / 64) for j in range(64)], 1.0),
    "pairs_part": (dict(theta=1e4, dim=64, interleaved=True), [1e4 ** (-j / 32) for j in range(32)], 1.0),
    "pairs_few": (dict(theta=1e4, dim=4, interleaved=True), [1.0, 0.01], 1.0),
    "part": (dict(theta=1e5, dim=96), [1e5 ** (-j / 48) for j in range(48)], 1.0),
    "few": (dict(theta=1e4, dim=4), [1.0, 0.01], 1.0),
    "odd": (dict(theta=1e4, dim=52), [1e4 ** (-j / 26) for j in range(26)], 1.0),
    "linear": (dict(theta=1e6, scaling="linear", factor=4.0), [1e6 ** (-j / 64) / 4 for j in range(64)], 1.0),
    "yarn": (dict(theta=1e6, scaling="yarn", factor=4.0, original=32768), yarn(1e6, 128, 4.0, 32768),
             0.1 * math.log(4) + 1),
    "yarn_part": (dict(theta=1e4, dim=64, scaling="yarn", factor=8.0, original=2048, gain=1.5, interleaved=True),
                  yarn(1e4, 64, 8.0, 2048), 1.5),
    "yarn_short": (dict(theta=1e6, scaling="yarn", factor=2.0, original=5), yarn(1e6, 128, 2.0, 5),
                   0.1 * math.log(2) + 1),
    "given": (dict(dim=8, freq=[0.5, 0.0, -0.25, 3.0], gain=2.0), [0.5, 0.0, -0.25, 3.0], 2.0),
}


def turned(x, w, pos, name, eps=1e-6):
    """Norm and rotation in binary64, and the bound's gain (|y| + |z|)."""
    args, freq, gain = ROPES[name]
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    size = x.abs() * max(gain, 1.0)
    a = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = gain * a.cos(), gain * a.sin()
    half = len(freq)
    first = torch.arange(half, device=x.device) * (2 if args.get("interleaved") else 1)
    second = first + (1 if args.get("interleaved") else half)
    y, z = x[..., first], x[..., second]
    x, size = x.clone(), size.clone()
    x[..., first], x[..., second] = y * c - z * s, y * s + z * c
    size[..., first] = size[..., second] = max(gain, 1.0) * (y.abs() + z.abs())
    return x, size


def check_turned(got, x, w, pos, name, dtype):
    o, size = turned(x, w, pos, name)
    tol = 28 * U * size
    if dtype == BF16:
        tol = tol + H * (o.abs() + tol)
    assert ((got.double() - o).abs() <= tol + 1e-30).all()


@pytest.mark.parametrize("io,cache_t,out_t", [(F32, F32, F32), (BF16, BF16, F32), (F32, BF16, BF16)])
@pytest.mark.parametrize("name", sorted(ROPES))
def test_rotations(q3, name, io, cache_t, out_t):
    """Every form of rotation, at positions from 0 to far beyond the trained ones; padding and rows behind the last."""
    from metalqwen3_b200.q3cu import Rope
    heads, n_kv, rows, lens = 12, 4, [37, 1, 9], [37, 300, 5]
    p = Paged(lens, n_kv, 16, cache_t, seed=1, fill=3.0)
    total = sum(rows)
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((total + 2, heads + 2 * n_kv, 128), generator=g, device="cuda").to(io)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:]
    qn, kn = (1 + 0.2 * torch.randn(128, generator=g, device="cuda") for _ in range(2))
    cache, batch = p.handles(offsets(rows))
    out = torch.full((total + 2, heads, 128), 9.0, dtype=out_t, device="cuda")
    rope = Rope(**ROPES[name][0])
    q3.kv_append(cache, batch, q, k, v, qn, kn, q_out=out, rope=rope)
    first = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        pad = max(0, r - n)
        span, pos = slice(first + pad, first + r), torch.arange(n - r + pad, n, device="cuda")
        assert (out[first:first + pad] == 9.0).all()
        first += r
        page_id, slot = p.where(s, pos)
        check_turned(out[span], q[span], qn, pos, name, out_t)
        check_turned(p.k[page_id, :, slot], k[span], kn, pos, name, cache_t)
        assert torch.equal(p.v[page_id, :, slot], v[span].to(cache_t))
    assert (out[total:] == 9.0).all()
    # without norms, in place
    dense = q.contiguous()
    if io == out_t:
        work = dense.clone()
        q3.kv_append(cache, batch, work, k, v, q_out=work, rope=rope)
        check_turned(work[37:38], dense[37:38], None, torch.tensor([299], device="cuda"), name, out_t)
    assert q3.device_status() == 0


def test_far_positions(q3):
    """Scaled and interleaved rotation past 2,000,000."""
    from metalqwen3_b200.q3cu import Rope
    page, pos = 256, 2_000_003
    for name in ("yarn", "pairs_part", "linear"):
        p = Paged([1], 2, page, F32, seed=3)
        p.table = torch.full((1, 8192), 1 << 30, dtype=torch.int32, device="cuda")
        p.table[0, pos // page] = 2
        p.kv_len[0] = pos + 1
        q, k, v = (queries(1, 2, F32, s) for s in (4, 5, 6))
        out = q3.kv_append(*p.handles([0, 1]), q, k, v, rope=Rope(**ROPES[name][0]))
        check_turned(out, q, None, torch.tensor([pos], device="cuda"), name, F32)
        check_turned(p.k[2, :, pos % page][None], k, None, torch.tensor([pos], device="cuda"), name, F32)
    assert q3.device_status() == 0


def test_default_rope_is_the_plain_append(q3):
    """A Rope of theta alone: the same bits as without one."""
    from metalqwen3_b200.q3cu import Rope
    p = Paged([70], 2, 16, F32, seed=5)
    q, k, v = (queries(70, h, F32, s) for h, s in ((6, 6), (2, 7), (2, 8)))
    cache, batch = p.handles([0, 70])
    a = q3.kv_append(cache, batch, q, k, v, theta=5e5)
    keys = p.k.clone()
    b = q3.kv_append(cache, batch, q, k, v, rope=Rope(theta=5e5))
    assert torch.equal(a, b) and torch.equal(keys.nan_to_num(0), p.k.nan_to_num(0))


def test_elements_that_are_not_turned_keep_infinities(q3):
    """Infinities in the elements behind the rotated ones (and rotated ones beside them) make no NaN elsewhere."""
    from metalqwen3_b200.q3cu import Rope
    for inter in (False, True):
        p = Paged([4], 1, 16, F32, seed=5)
        q, k, v = (queries(4, 1, F32, s) for s in (6, 7, 8))
        q[:, :, 100], q[:, :, 127] = math.inf, -math.inf
        out = q3.kv_append(*p.handles([0, 4]), q, k, v, rope=Rope(dim=64, interleaved=inter))
        assert torch.isfinite(out[..., :100]).all() and torch.equal(out[..., 64:], q[..., 64:])


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("name", ["plain", "halves", "pairs", "pairs_part", "part", "odd", "few", "yarn"])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [
    (32, 8, 64, [1], [4096]), (16, 8, 16, [1, 1, 1], [1, 17, 300]), (5, 5, 32, [3, 0, 33], [3, 0, 64]),
    (16, 1, 256, [70], [70]), (12, 4, 16, [9, 5], [4, 5]),
])
def test_append_quantised(q3, io, name, heads, n_kv, page, rows, lens):
    """Codes and scales are q3cu_quantize_q8's of the rows that an f32 cache gets; nothing else of the pool changes."""
    from metalqwen3_b200.q3cu import Rope
    total = sum(rows)
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((total + 2, heads + 2 * n_kv, 128), generator=g, device="cuda")
    qkv[:, :, 5::50] *= 6.0
    qkv[0, -1, :64] = 0.0                       # a group of zeros
    qkv[0, -1, 64:] *= 1e-40                    # and one of the least numbers
    qkv = qkv.to(io)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:]
    qn, kn = (1 + 0.2 * torch.randn(128, generator=g, device="cuda") for _ in range(2))
    rope = None if name == "plain" else Rope(**ROPES[name][0])
    wide = Paged(lens, n_kv, page, F32, seed=1, fill=3.0)
    p = Quantised(lens, n_kv, page, seed=1, gap=64, scale=-1.0)
    before = [t.clone() for t in p.pool + p.scale_pool]
    q_wide = q3.kv_append(*wide.handles(offsets(rows)), q, k, v, qn, kn, rope=rope, out_dtype=BF16)
    cache, batch = p.handles(offsets(rows))
    q_out = q3.kv_append(cache, batch, q, k, v, qn, kn, rope=rope)
    mine = torch.zeros(total + 2, dtype=torch.bool, device="cuda")
    assert q_out.dtype == BF16
    first = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        pad = max(0, r - n)
        mine[first + pad:first + r] = True
        first += r
        if r == pad:
            continue
        pos = range(n - r + pad, n)
        page_id, slot = p.where(s, pos)
        for side, (codes, scales) in zip((wide.k, wide.v), ((p.k, p.ks), (p.v, p.vs))):
            x = side[page_id, :, slot]
            want, step = q3.quantize_q8(x.reshape(-1, 128).contiguous())
            assert torch.equal(codes[page_id, :, slot].reshape(-1, 128), want)
            assert torch.equal(scales[page_id, :, slot].reshape(-1, 2), step)
            codes[page_id, :, slot], scales[page_id, :, slot] = 77, -1.0
    assert torch.equal(q_out[mine], q_wide[mine])
    for now, was in zip(p.pool + p.scale_pool, before):
        assert torch.equal(now, was)
    assert q3.device_status() == 0


def test_append_quantised_odd_values(q3):
    """NaN and infinities as in q3cu_quantize_q8: a NaN element is code 0, an infinity makes its group's scale infinite."""
    p = Quantised([3], 2, 16, seed=4)
    x = queries(3, 2, F32, 5)
    x[0, 0, 3], x[1, 1, 70], x[2, 0, 64:] = math.nan, math.inf, math.nan
    q3.kv_append(*p.handles([0, 3]), None, x, x)
    page, slot = p.where(0, range(3))
    want, step = q3.quantize_q8(x.reshape(-1, 128).contiguous())
    assert torch.equal(p.v[page, :, slot].reshape(-1, 128), want)
    assert torch.equal(p.vs[page, :, slot].reshape(-1, 2), step)


# ---- reading back --------------------------------------------------------------------------------

@pytest.mark.parametrize("cache_t", [F32, BF16, I8])
@pytest.mark.parametrize("out_t", [F32, BF16])
@pytest.mark.parametrize("n_kv,page,rows,lens", [
    (8, 16, [1], [4000]), (2, 64, [70, 0, 3, 1000], [70, 5, 300, 1000]), (17, 32, [9, 40], [4, 41]), (1, 256, [600], [600]),
])
def test_read(q3, cache_t, out_t, n_kv, page, rows, lens):
    """Rows of whole sequences and of their ends, padding as zeros, rows behind the last untouched; outputs with a stride."""
    p = (Quantised(lens, n_kv, page, seed=8, gap=32) if cache_t == I8 else Paged(lens, n_kv, page, cache_t, seed=8, gap=32)).fill(9)
    total = sum(rows)
    wide = torch.full((total + 2, 2 * n_kv + 1, 128), 9.0, dtype=out_t, device="cuda")
    k, v = wide[:, :n_kv], wide[:, n_kv + 1:]
    assert q3.kv_read(*p.handles(offsets(rows)), k_out=k, v_out=v)[0] is k
    assert (wide[:, n_kv] == 9.0).all() and (wide[total:] == 9.0).all()
    first = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        pad = max(0, r - n)
        assert (k[first:first + pad] == 0).all() and (v[first:first + pad] == 0).all()
        pos = range(n - r + pad, n)
        page_id, slot = p.where(s, pos)
        want = p.held(s, pos) if cache_t == I8 else (p.k[page_id, :, slot], p.v[page_id, :, slot])
        for got, w in zip((k, v), want):
            assert torch.equal(got[first + pad:first + r], w.to(out_t))
        first += r
    dense = q3.kv_read(*p.handles(offsets(rows)), rows=total, dtype=out_t)
    assert torch.equal(dense[0], k[:total]) and torch.equal(dense[1], v[:total])
    assert q3.device_status() == 0


def test_read_bad_pages(q3):
    """A page id outside the cache and a position behind the table: flagged, zeros; the other sequences are read."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    for bad in (-1, 1 << 30, None):
        p = Quantised([20, 20], 2, 16, seed=7, spare=1).fill(8)
        if bad is None:
            p.kv_len[0] = 1000
        else:
            p.table[0, 1] = bad
        k, v = q3.kv_read(*p.handles([0, 2, 4]), rows=4, dtype=F32)
        assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
        assert (k[:2] == 0).all() and (v[:2] == 0).all()
        want = p.held(1, [18, 19])
        assert torch.equal(k[2:], want[0]) and torch.equal(v[2:], want[1])


def test_far_pages_pass_32_bits(q3):
    """Codes beyond 2^31 bytes and scales beyond 2^31 bytes of their pools."""
    from metalqwen3_b200.q3cu import KVBatch, KVCache
    n_kv, page, far = 1, 16, 9
    pitch, sp = 1 << 28, 1 << 26
    codes = [torch.zeros((far + 1) * pitch, dtype=I8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((far + 1) * sp, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((far + 1, n_kv, page, 128), (pitch, page * 128, 128, 1)) for t in codes)
    ks, vs = (t.as_strided((far + 1, n_kv, page, 2), (sp, page * 2, 2, 1)) for t in scales)
    cache = KVCache(k, v, ks, vs)
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = KVBatch(torch.tensor([16], **i32), torch.tensor([[far]], **i32), torch.tensor([0, 16], **i32))
    x = queries(16, 1, F32, 3)
    q3.kv_append(cache, batch, None, x, x)
    back = q3.kv_read(cache, batch, rows=16, dtype=F32)
    want, step = q3.quantize_q8(x.reshape(-1, 128).contiguous())
    assert torch.equal(back[1].reshape(-1, 2, 64), want.float().reshape(-1, 2, 64) * step[..., None])
    assert torch.equal(v[far, 0], want) and torch.equal(vs[far, 0], step)
    assert q3.device_status() == 0


def test_append_and_read_as_a_graph_on_another_stream(q3):
    """Captured on a stream of its own and replayed while the sequence grows, eager calls on the current one between."""
    from metalqwen3_b200.q3cu import Rope
    p = Quantised([40], 2, 16, seed=6, scale=0.0)
    p.kv_len[0] = 1
    cache, batch = p.handles([0, 1])
    x, back = queries(1, 2, F32, 7), [torch.empty((1, 2, 128), device="cuda") for _ in range(2)]
    rope, stream = Rope(interleaved=True), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        q3.kv_append(cache, batch, None, x, x, rope=rope)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            q3.kv_append(cache, batch, None, x, x, rope=rope)
            q3.kv_read(cache, batch, k_out=back[0], v_out=back[1])
    for n in (1, 5, 40):
        x.copy_(queries(1, 2, F32, n))
        p.kv_len[0] = n
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, step = q3.quantize_q8(x.reshape(-1, 128).contiguous())
        assert torch.equal(back[1].reshape(-1, 2, 64), want.float().reshape(-1, 2, 64) * step[..., None])
        assert torch.equal(back[0], p.held(0, [n - 1])[0])
    assert q3.device_status() == 0
