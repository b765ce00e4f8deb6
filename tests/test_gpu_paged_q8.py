"""Attention over a Q8_0 paged cache against the formula in binary64 over the products of codes and scales.

Tolerances as in test_gpu_paged.py.  What is different here stays within their terms: f32 queries and weights are two f16
parts (2 u each), sums of products of codes are exact up to the tensor cores' cut (2 u a step of 16, 8 steps), scales are
one rounding each.  An f16 part is no finer than 2^-25, half its least number, and the largest query element of a row (the
largest value scale of 32 positions) is lifted to 2^14 or more, so that an element is also off by up to 2^-39 of the row's
largest: a score by 128 * 2^-39 max|q| max|k| / sqrt(128), a result of n positions by n 2^-39 (128 / 127) max|v|.
Where the result is bf16 a weight is one f16 part: 2^-11 relative each, in prompts too.  Prompts round scales and then
products of code and scale to f16 on their way: their formula is taken over the rounded elements (in f16 after
multiplication by a power of two, so that the rounding is that of 11 bits at any size; what lies 2^-39 below the largest
is within the terms above).  Their probabilities are no finer than 2^-25 where the largest are 2^7 to 2^15:
n 2^-32 max|v| for values of one size.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv_forms import I8, Quantised
from test_gpu_paged import BF16, DECODE, F32, H, PROMPT, U, attend, offsets, queries

pytestmark = pytest.mark.gpu
W = 2.0 ** -11


def check_attention(got, q, k, v, seen, dtype, weight_rounding=0.0, floor=2.0 ** -39):
    o, pv, a = attend(q.double(), k, v, seen)
    n, top = max(1, k.shape[0]), lambda x: float(x.abs().max()) if x.numel() else 0.0
    ds = 160 * U * a + math.sqrt(128) * 2.0 ** -39 * top(q) * top(k)
    tol = (torch.expm1(2 * ds) + (n + 64) * U + weight_rounding) * pv + n * floor * 1.01 * top(v)
    if dtype == BF16:
        tol = tol + H * (o.abs() + tol)
    bad = ~((got.double() - o).abs() <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - o).abs().max()),
                           float(tol.max()))


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("heads,n_kv,page,lens", DECODE + [(10, 2, 256, [127, 128, 129, 255, 256, 257, 700]),
                                                           (3, 1, 128, [33, 95, 96, 97, 4000])])
def test_attention_paged(q3, io, heads, n_kv, page, lens):
    p = Quantised(lens, n_kv, page, seed=11).fill(12)
    q = queries(len(lens), heads, io, 13)
    cache, batch = p.handles()
    got = q3.attention_paged(cache, batch, q)
    for s, n in enumerate(lens):
        k, v = p.rows(s)
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [n], io, W if io == BF16 else 0.0)
    assert q3.device_status() == 0


def test_attention_paged_peaked_flat_and_uneven(q3):
    """Scores in the thousands, all equal, queries and scales far from 1, and scales that differ by 10^6 within a tile."""
    for scale, size in ((60.0, 1.0), (0.0, 1.0), (1e-12, 1e9), (1e15, 1e-14)):
        p = Quantised([777, 64], 2, 16, seed=14).fill(15, size)
        q = queries(2, 8, F32, 16, scale)
        got = q3.attention_paged(*p.handles(), q)
        for s, n in enumerate(p.lens):
            check_attention(got[s:s + 1], q[s:s + 1], *p.rows(s), [n], F32)
    p = Quantised([300], 2, 16, seed=14).fill(15)
    page, slot = p.where(0, range(0, 300, 3))
    p.vs[page, :, slot] *= 1e-6
    p.ks[page, :, slot] *= 1e-3
    q = queries(1, 8, F32, 16)
    check_attention(q3.attention_paged(*p.handles(), q), q, *p.rows(0), [300], F32)


def test_attention_paged_strides_and_work(q3):
    """Pages (and their scales) further apart than they are large; queries inside wider rows; any workspace contents."""
    p = Quantised([100, 257, 0], 4, 32, seed=17, gap=4096 + 32).fill(18)
    wide = queries(3, 24, F32, 19)
    q = wide[:, 4:12]
    cache, batch = p.handles()
    out = torch.empty((3, 8, 128), device="cuda")
    work = torch.full((q3.attention_paged_workspace(cache, 8).numel(),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert q3.attention_paged(cache, batch, q, out=out, work=work) is out
        for s, n in enumerate(p.lens):
            check_attention(out[s:s + 1], q[s:s + 1], *p.rows(s), [n], F32)


def test_attention_paged_bad_pages(q3):
    """Bad page ids read as zeros and are flagged; a length beyond the table is cut; a negative one is empty."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    p = Quantised([100, 40, 50, 50], 2, 16, seed=20).fill(21)
    k, v = p.rows(0)
    for i, bad in ((1, -3), (4, p.n_pages)):
        p.table[0, i] = bad
        k[16 * i:16 * i + 16] = 0
        v[16 * i:16 * i + 16] = 0
    cap = p.max_pages * 16
    p.table[2] = p.table[0, 0]                  # one page many times over: a full table row
    p.kv_len[2], p.kv_len[3] = cap + 1, -5
    q = queries(4, 4, F32, 22)
    got = q3.attention_paged(*p.handles(), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    check_attention(got[:1], q[:1], k, v, [100], F32)
    check_attention(got[1:2], q[1:2], *p.rows(1), [40], F32)
    again = torch.arange(cap, device="cuda") % 16
    page = p.table[0, 0].long()
    kk, vv = ((t[page].double() * c[page].double().repeat_interleave(64, -1)).transpose(0, 1)[again]
              for t, c in ((p.k, p.ks), (p.v, p.vs)))
    check_attention(got[2:3], q[2:3], kk, vv, [cap], F32)
    assert (got[3] == 0).all()


@pytest.mark.parametrize("io", [F32, BF16])
def test_appended_and_attended_as_a_graph(q3, io):
    """A serving step's append and attention, captured and replayed while the sequences grow."""
    lens, heads, n_kv = [5, 130, 31], 8, 2
    p = Quantised([n + 40 for n in lens], n_kv, 16, seed=30).fill(31)
    qkv = queries(3, heads + 2 * n_kv, F32, 32)
    cache, batch = p.handles([0, 1, 2, 3])
    work, out = q3.attention_paged_workspace(cache, heads), torch.empty((3, heads, 128), dtype=io, device="cuda")
    q_out = torch.empty_like(out)

    def step():
        q3.kv_append(cache, batch, qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:], q_out=q_out)
        q3.attention_paged(cache, batch, q_out, out=out, work=work)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for n in (1, 7, 40):
        now = [x + n for x in lens]
        p.kv_len.copy_(torch.tensor(now, dtype=torch.int32))
        qkv.copy_(queries(3, heads + 2 * n_kv, F32, 33 + n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for s, x in enumerate(now):
            p.lens = now
            check_attention(out[s:s + 1], q_out[s:s + 1], *p.rows(s), [x], io, W if io == BF16 else 0.0)
    assert q3.device_status() == 0


def test_unused_scales_and_nan(q3):
    """NaN scales behind the length (there everywhere: the pool is full of them) reach nothing; one at a value of the
    sequence reaches its 64 elements only, one at a key its head only."""
    p = Quantised([100, 50], 2, 16, seed=40).fill(41)
    q = queries(2, 4, F32, 42)
    clean = q3.attention_paged(*p.handles(), q)
    assert torch.isfinite(clean).all()
    page, slot = p.where(0, [70])
    p.vs[page, 1, slot, 1] = math.nan
    got = q3.attention_paged(*p.handles(), q)
    assert torch.isnan(got[0, 2:, 64:]).all()
    assert torch.equal(got[0, 2:, :64], clean[0, 2:, :64]) and torch.equal(got[0, :2], clean[0, :2])
    assert torch.equal(got[1], clean[1])
    p.ks[page, 0, slot, 0] = math.nan
    got = q3.attention_paged(*p.handles(), q)
    assert torch.isnan(got[0, :2]).all() and torch.equal(got[1], clean[1])


# ---- prompts -----------------------------------------------------------------------------------

def rounded(p, s):
    """Keys and values of sequence s as the prompts' products take them."""
    page, slot = p.where(s, range(max(p.lens[s], 0)))
    out = []
    for t, c in ((p.k, p.ks), (p.v, p.vs)):
        scale = c[page, :, slot]
        top = float(scale.nan_to_num(0.0, 0.0, 0.0).abs().max()) if scale.numel() else 0.0
        up = 2.0 ** (14 - math.floor(math.log2(top))) if top else 1.0
        x = (scale * up).half().repeat_interleave(64, -1) * (t[page, :, slot].half() / 128)
        out.append(x.double() * (128 / up))
    return tuple(out)


@pytest.mark.parametrize("heads,n_kv,page,rows,lens", PROMPT + [(32, 8, 64, [3], [7000]), (8, 1, 16, [100, 20], [2500, 3000])])
def test_attention_prompt(q3, heads, n_kv, page, rows, lens):
    """Whole prompts, chunks behind a prefix (few rows behind a long one share an item), rows that see nothing, rows behind
    the last sequence."""
    p = Quantised(lens, n_kv, page, seed=31).fill(32)
    total = sum(rows)
    q = queries(total + 3, heads, BF16, 33)
    out = torch.full((total + 3, heads, 128), 7.0, dtype=BF16, device="cuda")
    assert q3.attention_prompt(*p.handles(offsets(rows)), q, out=out) is out
    assert (out[total:] == 7.0).all()
    first = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        if r:
            check_attention(out[first:first + r], q[first:first + r], *rounded(p, s), [max(0, n - r + 1 + i) for i in range(r)],
                            BF16, W, 2.0 ** -32)
        first += r
    assert q3.device_status() == 0


@pytest.mark.parametrize("n_seqs", [33, 100])
def test_attention_prompt_many_sequences(q3, n_seqs):
    g = np.random.default_rng(n_seqs)
    rows = [int(r) if r < 40 or i % 9 == 0 else int(r) % 40 for i, r in enumerate(g.integers(0, 300, n_seqs))]
    lens = [r + int(x) for r, x in zip(rows, g.integers(0, 400, n_seqs) * g.integers(0, 2, n_seqs))]
    p = Quantised(lens, 2, 16, seed=47).fill(48)
    off = offsets(rows)
    q = queries(off[-1], 4, BF16, 49)
    out = q3.attention_prompt(*p.handles(off), q)
    for s in range(n_seqs):
        if rows[s]:
            mine = slice(off[s], off[s + 1])
            check_attention(out[mine], q[mine], *rounded(p, s), range(lens[s] - rows[s] + 1, lens[s] + 1), BF16, W, 2.0 ** -32)
    assert q3.device_status() == 0


def test_attention_prompt_long(q3):
    """Many items to a CTA, and many key tiles to an item; strides, bad pages."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    n = 2500
    p = Quantised([n], 4, 16, seed=40, gap=4096 + 32).fill(41)
    k, v = rounded(p, 0)
    for i, bad in ((2, -1), (9, 1 << 30)):
        p.table[0, i] = bad
        k[16 * i:16 * i + 16] = 0
        v[16 * i:16 * i + 16] = 0
    q = queries(n, 48, BF16, 42)[:, 8:40]
    got = q3.attention_prompt(*p.handles([0, n]), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    some = list(range(0, n, 97)) + [n - 1]
    check_attention(got[some], q[some], k, v, [i + 1 for i in some], BF16, W, 2.0 ** -32)


def test_attention_prompt_hides_later_rows(q3):
    """NaN and infinite scales at later positions reach no earlier row; what a row sees of them it shows."""
    n = 150
    for rows in (n, 3):                         # a prompt, and its last rows alone
        p = Quantised([n], 2, 16, seed=34).fill(35)
        page, slot = p.where(0, range(n))
        for at, what in ((147, math.nan), (148, math.inf)):
            p.vs[page[at], :, slot[at], 1] = what
            p.ks[page[at], 1, slot[at], 0] = what
        q = queries(rows, 8, BF16, 36)
        got = q3.attention_prompt(*p.handles([0, rows]), q)
        k, v = (t[:147] for t in rounded(p, 0))
        early = rows - 3
        if early:
            check_attention(got[:early], q[:early], k, v, range(1, early + 1), BF16, W, 2.0 ** -32)
        assert torch.isnan(got[early:, :4, 64:]).all() and torch.isnan(got[early:, 4:]).all()
        assert torch.isfinite(got[early, :4, :64]).all()


def test_attention_prompt_peaked_and_flat(q3):
    for scale in (40.0, 0.0):
        p = Quantised([333], 2, 32, seed=37).fill(38, scale if scale else 1.0)
        q = queries(333, 8, BF16, 39, scale)
        check_attention(q3.attention_prompt(*p.handles([0, 333]), q), q, *rounded(p, 0), range(1, 334), BF16, W, 2.0 ** -32)


def test_attention_prompt_uneven_scales(q3):
    """Values and keys of very different sizes: tiles of larger values after smaller ones and the other way round; within a
    tile, a later position 2^40 times larger takes no bits from earlier rows."""
    n = 600
    g = torch.Generator(device="cuda").manual_seed(60)
    for sizes in ([2.0 ** (i // 128 * 3) for i in range(n)], [2.0 ** -(i // 128 * 3) for i in range(n)],
                  [2.0 ** (i % 7) for i in range(n)]):
        p = Quantised([n], 2, 16, seed=61).fill(62)
        page, slot = p.where(0, range(n))
        f = torch.tensor(sizes, device="cuda")
        p.vs[page, :, slot] *= f[:, None, None]
        p.ks[page, :, slot] *= torch.rand((n, 1, 1), generator=g, device="cuda") * 0.9 + 0.1
        q = queries(n, 8, BF16, 63)
        got = q3.attention_prompt(*p.handles([0, n]), q)
        # as far as the rows see: a value's part of the error is relative to the largest it may be summed with
        for a, b in ((0, 128), (128, 300), (300, n)):
            check_attention(got[a:b], q[a:b], *(t[:b] for t in rounded(p, 0)), range(a + 1, b + 1), BF16, W, 2.0 ** -32)
    for rows in (n, 5):
        p = Quantised([n], 2, 16, seed=64).fill(65)
        page, slot = p.where(0, range(n))
        clean = q3.attention_prompt(*p.handles([0, rows]), q[:rows])
        p.vs[page[n - 2], :, slot[n - 2]] *= 2.0 ** 40
        p.ks[page[n - 1], :, slot[n - 1]] *= 2.0 ** 40
        got = q3.attention_prompt(*p.handles([0, rows]), q[:rows])
        check_attention(got[:rows - 2], q[:rows - 2], *(t[:n - 2] for t in p.rows(0)),
                        range(n - rows + 1, n - 1), BF16, 2.0 ** -8)
        assert torch.isfinite(clean).all()
    assert q3.device_status() == 0


def test_attention_prompt_sizes(q3):
    """Queries, keys and values far from 1."""
    for size_q, size_kv in ((1e-6, 1e6), (1e8, 1e-8), (1.0, 1e-20), (1e20, 1e-20), (1e-30, 1.0)):
        p = Quantised([300], 2, 16, seed=66).fill(67, size_kv)
        q = queries(300, 8, BF16, 68, size_q)
        got = q3.attention_prompt(*p.handles([0, 300]), q)
        check_attention(got, q, *rounded(p, 0), range(1, 301), BF16, W, 2.0 ** -32)
    assert q3.device_status() == 0
