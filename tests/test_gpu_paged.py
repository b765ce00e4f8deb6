"""The paged-cache operators (q3cu_kv_append, q3cu_attention_paged,
q3cu_attention_prompt) against their formulas in binary64.

Tolerances, per output element, from the roundings the operators make
(u = 2^-24, half a step of binary32; H = 2^-8, half a step of bf16):
  * a score is a 128-term dot product: off by at most (128 + 32) u A with
    A = sum |q_i k_i| / sqrt(128), the 32 covering the scale, the exponent's
    product and products of split operands (2^-21 each); a softmax weight is
    then off by a factor e^(2 ds), and the weighted sum of n values by another
    (n + 64) u;
  * the bf16 prompt path rounds every probability to bf16: H relative each;
  * a bf16 result is rounded once: H |o|.
  * rotation: a tree sum of 128 squares, a root, a division and two products
    are within 16 u, sine and cosine within 4 u: 24 u (|y_j| + |y_{j+64}|).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


class Paged:
    """A pool of pages full of NaN, and sequences laid out on shuffled pages of it."""

    def __init__(self, lens, n_kv, page, dtype, seed, spare=3, gap=0, fill=NAN):
        self.lens, self.n_kv, self.page, self.dtype = list(lens), n_kv, page, dtype
        g = torch.Generator().manual_seed(seed)
        used = [(max(n, 0) + page - 1) // page for n in lens]
        self.n_pages = sum(used) + spare
        pitch = n_kv * page * 128 + gap
        self.pool = [torch.full((self.n_pages, pitch), fill, dtype=dtype, device="cuda") for _ in range(2)]
        self.k, self.v = (p.as_strided((self.n_pages, n_kv, page, 128), (pitch, page * 128, 128, 1)) for p in self.pool)
        ids = torch.randperm(self.n_pages, generator=g)
        self.max_pages = max(max(used), 1) + 2
        table = torch.full((len(lens), self.max_pages), -7, dtype=torch.int32)
        a = 0
        for s, n in enumerate(used):
            table[s, :n] = ids[a:a + n].int()
            a += n
        self.table = table.cuda()
        self.kv_len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def where(self, s, positions):
        p = torch.as_tensor(positions, device="cuda").long()
        return self.table[s][p // self.page].long(), p % self.page

    def fill(self, seed, scale=1.0):
        """Random keys and values at every position of every sequence."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        for s, n in enumerate(self.lens):
            if n > 0:
                page, slot = self.where(s, range(n))
                for t in (self.k, self.v):
                    x = torch.randn((n, self.n_kv, 128), generator=g, device="cuda") * scale
                    t[page, :, slot] = x.to(self.dtype)
        return self

    def rows(self, s):
        """Keys and values of sequence s, [n][n_kv][128], binary64."""
        page, slot = self.where(s, range(max(self.lens[s], 0)))
        return self.k[page, :, slot].double(), self.v[page, :, slot].double()

    def handles(self, row_off=None):
        from metalqwen3_b200.q3cu import KVBatch, KVCache
        off = None if row_off is None else torch.tensor(row_off, dtype=torch.int32, device="cuda")
        return KVCache(self.k, self.v), KVBatch(self.kv_len, self.table, off)


def offsets(rows):
    return [0] + list(np.cumsum(rows).astype(int))


def attend(q, k, v, seen):
    """q [r][heads][128], k and v [n][n_kv][128] (binary64); row i sees the first seen[i] keys.
    Returns (o, sum p|v|, max A over the seen keys)."""
    r, heads, _ = q.shape
    n, n_kv, _ = k.shape
    o = torch.zeros((r, heads, 128), dtype=torch.float64, device=q.device)
    pv, amax = o.clone(), torch.zeros((r, heads, 1), dtype=torch.float64, device=q.device)
    seen = torch.as_tensor(seen, device=q.device)
    for h in range(heads):
        kk, vv = k[:, h // (heads // n_kv)], v[:, h // (heads // n_kv)]
        hidden = torch.arange(n, device=q.device)[None] >= seen[:, None]
        kc = torch.where(torch.isfinite(kk), kk, torch.zeros_like(kk))
        s = torch.where(hidden, -math.inf, q[:, h] @ kk.T / math.sqrt(128))
        a = torch.where(hidden, 0.0, q[:, h].abs() @ kc.abs().T / math.sqrt(128))
        live = seen > 0
        p = torch.zeros_like(s)
        p[live] = torch.softmax(s[live], -1)
        for i in range(r):                      # only the seen values: 0 * NaN is not 0
            m = int(min(max(int(seen[i]), 0), n))
            if m:
                o[i, h], pv[i, h] = p[i, :m] @ vv[:m], p[i, :m] @ vv[:m].abs()
        if n:
            amax[:, h, 0] = a.amax(-1)
    return o, pv, amax


def check_attention(got, q, k, v, seen, dtype, prob_rounding=0.0):
    o, pv, a = attend(q.double(), k, v, seen)
    n = max(1, k.shape[0])
    tol = (torch.expm1(2 * 160 * U * a) + (n + 64) * U + prob_rounding) * pv
    if dtype == BF16:
        tol = tol + H * (o.abs() + tol)
    bad = ~((got.double() - o).abs() <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - o).abs().max()),
                           float(tol.max()))


def queries(rows, heads, dtype, seed, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, heads, 128), generator=g, device="cuda") * scale).to(dtype)


# ---- append ------------------------------------------------------------------------------------

def rotated(x, w, pos, eps=1e-6, theta=1e6):
    """Norm (with weights) and rotation in binary64; also |y_j| + |y_{j+64}|."""
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    a = pos.double()[:, None, None] * theta ** (-torch.arange(64, dtype=torch.float64, device=x.device) / 64)
    y, z = x[..., :64], x[..., 64:]
    size = (y.abs() + z.abs()).repeat(1, 1, 2)
    return torch.cat([y * a.cos() - z * a.sin(), y * a.sin() + z * a.cos()], -1), size


def check_rotated(got, x, w, pos, dtype):
    o, size = rotated(x, w, pos)
    tol = 24 * U * size
    if dtype == BF16:
        tol = tol + H * (o.abs() + tol)
    assert ((got.double() - o).abs() <= tol).all()


@pytest.mark.parametrize("io,cache_t,out_t", [(F32, BF16, BF16), (F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32),
                                              (F32, BF16, F32)])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [
    (32, 8, 64, [1], [4096]), (16, 8, 16, [1, 1, 1], [1, 17, 300]), (40, 8, 128, [37, 1, 260], [37, 500, 1000]),
    (5, 5, 32, [3, 0, 33], [3, 0, 64]), (16, 1, 256, [70], [70]), (12, 4, 16, [9, 5], [4, 5]),
])
def test_append(q3, io, cache_t, out_t, heads, n_kv, page, rows, lens):
    """Fused projection rows; two rows behind the last sequence; the sequence (9 rows, length 4) starts with padding."""
    p = Paged(lens, n_kv, page, cache_t, seed=1, fill=3.0)
    total = sum(rows)
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((total + 2, heads + 2 * n_kv, 128), generator=g, device="cuda").to(io)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:]
    qn, kn = (1 + 0.2 * torch.randn(128, generator=g, device="cuda") for _ in range(2))
    before = p.k.clone(), p.v.clone()
    out = torch.full((total + 2, heads, 128), 9.0, dtype=out_t, device="cuda")
    cache, batch = p.handles(offsets(rows))
    assert q3.kv_append(cache, batch, q, k, v, qn, kn, q_out=out) is out
    assert q3.device_status() == 0
    first, touched = 0, torch.zeros(p.k.shape, dtype=torch.bool, device="cuda")
    for s, (r, n) in enumerate(zip(rows, lens)):
        pad = max(0, r - n)
        span, pos = slice(first + pad, first + r), torch.arange(n - r + pad, n, device="cuda")
        assert (out[first:first + pad] == 9.0).all()
        first += r
        if r == pad:
            continue
        page_id, slot = p.where(s, pos)
        check_rotated(out[span], q[span], qn, pos, out_t)
        check_rotated(p.k[page_id, :, slot], k[span], kn, pos, cache_t)
        assert torch.equal(p.v[page_id, :, slot], v[span].to(cache_t))
        touched[page_id, :, slot] = True
    assert (out[total:] == 9.0).all()
    for now, was in zip((p.k, p.v), before):
        assert torch.equal(now[~touched], was[~touched])


def test_append_many_sequences(q3):
    """300 sequences of 0 to 3 rows: each row finds its own."""
    g = np.random.default_rng(5)
    rows = [int(r) for r in g.integers(0, 4, 300)]
    lens = [r + int(x) for r, x in zip(rows, g.integers(0, 200, 300))]
    p = Paged(lens, 2, 16, F32, seed=9, fill=0.0)
    off = offsets(rows)
    q, k, v = (queries(off[-1], 2, F32, s) for s in (10, 11, 12))
    out = q3.kv_append(*p.handles(off), q, k, v)
    for s in range(300):
        if rows[s]:
            mine, pos = slice(off[s], off[s + 1]), torch.arange(lens[s] - rows[s], lens[s], device="cuda")
            page_id, slot = p.where(s, pos)
            check_rotated(out[mine], q[mine], None, pos, F32)
            check_rotated(p.k[page_id, :, slot], k[mine], None, pos, F32)
            assert torch.equal(p.v[page_id, :, slot], v[mine])
    assert q3.device_status() == 0


def test_append_far_positions_no_norm_no_queries_in_place(q3):
    """Positions past 2,000,000 (pages before the row's are never read), the rotation alone, q_out = q, and keys and
    values alone."""
    page, pos = 256, 2_000_003
    p = Paged([1], 2, page, F32, seed=3)
    p.table = torch.full((1, 8192), 1 << 30, dtype=torch.int32, device="cuda")
    p.table[0, pos // page] = 2
    p.kv_len[0] = pos + 1
    q, k, v = (queries(1, 2, F32, s) for s in (4, 5, 6))
    cache, batch = p.handles([0, 1])
    work = q.clone()
    assert q3.kv_append(cache, batch, work, k, v, q_out=work) is work
    at = torch.tensor([pos], device="cuda")
    check_rotated(work, q, None, at, F32)
    check_rotated(p.k[2, :, pos % page][None], k, None, at, F32)
    p.k.fill_(0), p.v.fill_(0)
    q3.kv_append(cache, batch, None, k, v)
    check_rotated(p.k[2, :, pos % page][None], k, None, at, F32)
    assert torch.equal(p.v[2, :, pos % page][None], v)
    assert q3.device_status() == 0


def test_append_bad_pages_and_positions(q3):
    """A page id outside the cache, a position behind the table: flagged, nothing stored, the queries still rotated."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    for bad in (-1, 5, 1 << 30, None):
        p = Paged([20, 20], 2, 16, F32, seed=7, spare=1, fill=1.0)
        assert p.n_pages == 5
        if bad is None:
            p.kv_len[0] = 1000                  # beyond the table's pages
        else:
            p.table[0, 1] = bad
        q, k, v = (queries(2, 2, F32, s) for s in (4, 5, 6))
        cache, batch = p.handles([0, 1, 2])
        before = p.k.clone()
        q3.kv_append(cache, batch, q, k, v)
        assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
        page_id, slot = p.where(1, [19])
        check_rotated(p.k[page_id, :, slot], k[1:], None, torch.tensor([19], device="cuda"), F32)
        p.k[page_id, :, slot] = 1.0
        assert torch.equal(p.k, before)


# ---- one token per sequence --------------------------------------------------------------------

DECODE = [
    (16, 8, 16, [512]), (32, 8, 64, [0, 1, 15, 16, 17, 63, 64, 65, 129, 1000]), (40, 8, 128, [1]),
    (8, 8, 32, [300, 31, 33]), (64, 8, 16, [2049, 0, 0, 7]), (16, 1, 256, [1500, 3]), (12, 4, 16, [0]),
    (32, 8, 16, [5, 900] * 40), (4, 4, 64, [20011]),
]


@pytest.mark.parametrize("io,cache_t", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("heads,n_kv,page,lens", DECODE)
def test_attention_paged(q3, io, cache_t, heads, n_kv, page, lens):
    p = Paged(lens, n_kv, page, cache_t, seed=11).fill(12)
    q = queries(len(lens), heads, io, 13)
    cache, batch = p.handles()
    got = q3.attention_paged(cache, batch, q)
    for s, n in enumerate(lens):
        k, v = p.rows(s)
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [n], io)
    assert q3.device_status() == 0


@pytest.mark.parametrize("cache_t", [F32, BF16])
def test_attention_paged_peaked_and_flat(q3, cache_t):
    """Scores in the thousands (one key takes all), and all equal."""
    for scale in (60.0, 0.0):
        p = Paged([777, 64], 2, 16, cache_t, seed=14).fill(15, scale if scale else 1.0)
        q = queries(2, 8, F32, 16, scale)
        cache, batch = p.handles()
        got = q3.attention_paged(cache, batch, q)
        for s, n in enumerate(p.lens):
            check_attention(got[s:s + 1], q[s:s + 1], *p.rows(s), [n], F32)


@pytest.mark.parametrize("cache_t", [F32, BF16])
def test_attention_paged_strides(q3, cache_t):
    """Pages further apart than they are large; queries inside wider rows."""
    p = Paged([100, 257, 0], 4, 32, cache_t, seed=17, gap=4096 + 8).fill(18)
    wide = queries(3, 24, F32, 19)
    q = wide[:, 4:12]
    cache, batch = p.handles()
    out = torch.empty((3, 8, 128), device="cuda")
    work = torch.full((q3.attention_paged_workspace(cache, 8).numel(),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):                          # the workspace's contents do not matter
        assert q3.attention_paged(cache, batch, q, out=out, work=work) is out
        for s, n in enumerate(p.lens):
            check_attention(out[s:s + 1], q[s:s + 1], *p.rows(s), [n], F32)


@pytest.mark.parametrize("cache_t", [F32, BF16])
def test_attention_paged_bad_pages(q3, cache_t):
    """Bad page ids read as zeros and are flagged; a length beyond the table is cut; a negative one is empty."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    p = Paged([100, 40, 50, 50], 2, 16, cache_t, seed=20).fill(21)
    k, v = p.rows(0)
    for i, bad in ((1, -3), (4, p.n_pages)):
        p.table[0, i] = bad
        k[16 * i:16 * i + 16] = 0
        v[16 * i:16 * i + 16] = 0
    cap = p.max_pages * 16
    p.table[2] = p.table[0, 0]                  # one page many times over: a full table row
    p.kv_len[2], p.kv_len[3] = cap + 1, -5
    q = queries(4, 4, F32, 22)
    cache, batch = p.handles()
    got = q3.attention_paged(cache, batch, q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    check_attention(got[:1], q[:1], k, v, [100], F32)
    check_attention(got[1:2], q[1:2], *p.rows(1), [40], F32)
    again = torch.arange(cap, device="cuda") % 16
    page = p.table[0, 0].long()
    check_attention(got[2:3], q[2:3], p.k[page].double().transpose(0, 1)[again],
                    p.v[page].double().transpose(0, 1)[again], [cap], F32)
    assert (got[3] == 0).all()


def test_attention_paged_equals_one_token_attention(q3):
    """The same token through q3cu_attention's contiguous f32 cache."""
    n = 700
    p = Paged([n], 8, 16, F32, seed=23).fill(24)
    q = queries(1, 32, F32, 25)
    k, v = (t.float().reshape(n, 1024).contiguous() for t in p.rows(0))
    xb, _ = q3.attention(q[0], k, v, n - 1, 4)
    got = q3.attention_paged(*p.handles(), q)
    check_attention(xb[None], q, *p.rows(0), [n], F32)
    check_attention(got, q, *p.rows(0), [n], F32)


def test_far_pages_pass_32_bits(q3):
    """Page starts beyond 2^31 elements and 2^32 bytes, for all three operators."""
    gap = (1 << 30) + 1024
    p = Paged([40], 1, 16, BF16, seed=26, spare=0, gap=gap, fill=0.0)
    assert p.k.stride(0) * 2 * (p.n_pages - 1) > 1 << 32
    q, k, v = queries(40, 4, BF16, 27), queries(40, 1, BF16, 28), queries(40, 1, BF16, 29)
    cache, batch = p.handles([0, 40])
    rq = q3.kv_append(cache, batch, q, k, v)
    check_rotated(p.k[p.where(0, range(40))[0], :, p.where(0, range(40))[1]], k, None, torch.arange(40, device="cuda"), BF16)
    check_attention(q3.attention_prompt(cache, batch, rq), rq, *p.rows(0), range(1, 41), BF16, H)
    check_attention(q3.attention_paged(cache, batch, rq[39:]), rq[39:], *p.rows(0), [40], BF16)
    assert q3.device_status() == 0


# ---- prompts -----------------------------------------------------------------------------------

PROMPT = [
    (16, 8, 16, [37], [37]), (32, 8, 64, [1, 2, 129, 64], [1, 2, 129, 64]), (8, 8, 128, [300], [300]),
    (40, 8, 16, [26, 25, 51], [26, 25, 51]), (16, 1, 32, [50], [50]), (64, 8, 256, [17, 200], [400, 200]),
    (12, 4, 16, [43, 1, 0, 90], [300, 1025, 0, 90]), (32, 8, 16, [9, 40], [4, 0]), (16, 8, 64, [5, 130], [700, 1290]),
    (32, 8, 128, [1] * 70, list(range(70))),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", PROMPT)
def test_attention_prompt(q3, dtype, heads, n_kv, page, rows, lens):
    """Whole prompts, chunks behind a prefix, rows that see nothing (length below the rows), rows behind the last
    sequence."""
    p = Paged(lens, n_kv, page, dtype, seed=31).fill(32)
    total = sum(rows)
    q = queries(total + 3, heads, dtype, 33)
    cache, batch = p.handles(offsets(rows))
    out = torch.full((total + 3, heads, 128), 7.0, dtype=dtype, device="cuda")
    assert q3.attention_prompt(cache, batch, q, out=out) is out
    assert (out[total:] == 7.0).all()
    first = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        k, v = p.rows(s)
        seen = [max(0, n - r + 1 + i) for i in range(r)]
        if r:
            check_attention(out[first:first + r], q[first:first + r], k, v, seen, dtype, H if dtype == BF16 else 0.0)
        first += r
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n_seqs", [33, 50, 64, 65, 100])
def test_attention_prompt_many_sequences(q3, dtype, n_seqs):
    """More sequences than a warp has lanes, and than it sorts: rows of 0 to 300, prefixes of 0 to 400."""
    g = np.random.default_rng(n_seqs)
    rows = [int(r) if r < 40 or i % 9 == 0 else int(r) % 40 for i, r in enumerate(g.integers(0, 300, n_seqs))]
    lens = [r + int(x) for r, x in zip(rows, g.integers(0, 400, n_seqs) * g.integers(0, 2, n_seqs))]
    p = Paged(lens, 2, 16, dtype, seed=47).fill(48)
    off = offsets(rows)
    q = queries(off[-1], 4, dtype, 49)
    out = q3.attention_prompt(*p.handles(off), q)
    for s in range(n_seqs):
        if rows[s]:
            k, v = p.rows(s)
            mine = slice(off[s], off[s + 1])
            check_attention(out[mine], q[mine], k, v, range(lens[s] - rows[s] + 1, lens[s] + 1), dtype,
                            H if dtype == BF16 else 0.0)
    one = q3.attention_paged(*p.handles(), queries(n_seqs, 4, dtype, 50))
    for s in range(n_seqs):
        check_attention(one[s:s + 1], queries(n_seqs, 4, dtype, 50)[s:s + 1], *p.rows(s), [lens[s]], dtype)
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_prompt_hides_later_rows(q3, dtype):
    """NaN and infinities at a later position reach no earlier row."""
    n = 150
    p = Paged([n], 2, 16, dtype, seed=34).fill(35)
    page, slot = p.where(0, range(n))
    for at, what in ((90, NAN), (91, math.inf), (140, -math.inf)):
        p.k[page[at], 1, slot[at]] = what
        p.v[page[at], :, slot[at]] = what
    q = queries(n, 8, dtype, 36)
    got = q3.attention_prompt(*p.handles([0, n]), q)
    k, v = p.rows(0)
    check_attention(got[:90], q[:90], k[:90], v[:90], range(1, 91), dtype, H if dtype == BF16 else 0.0)
    assert torch.isnan(got[90:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("at", list(range(17)) + [127, 128, 190])
def test_nan_key_shows_in_every_row_that_sees_it(q3, dtype, at):
    """A NaN key, wherever it lies in a tile, in prompt rows and in single tokens; earlier rows stay as they are."""
    n = 200
    p = Paged([n], 1, 16, dtype, seed=56).fill(57)
    page, slot = p.where(0, range(n))
    p.k[page[at], :, slot[at]] = NAN
    q = queries(n, 4, dtype, 58)
    cache, batch = p.handles([0, n])
    got = q3.attention_prompt(cache, batch, q)
    assert torch.isnan(got[at:]).all() and torch.isfinite(got[:at]).all()
    assert torch.isnan(q3.attention_paged(cache, batch, q[:1])).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_prompt_peaked_and_flat(q3, dtype):
    for scale in (40.0, 0.0):
        p = Paged([333], 2, 32, dtype, seed=37).fill(38, scale if scale else 1.0)
        q = queries(333, 8, dtype, 39, scale)
        got = q3.attention_prompt(*p.handles([0, 333]), q)
        check_attention(got, q, *p.rows(0), range(1, 334), dtype, H if dtype == BF16 else 0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_prompt_strides_and_bad_pages(q3, dtype):
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    n = 200
    p = Paged([n], 2, 16, dtype, seed=40, gap=264).fill(41)
    k, v = p.rows(0)
    for i, bad in ((2, -1), (9, 1 << 30)):
        p.table[0, i] = bad
        k[16 * i:16 * i + 16] = 0
        v[16 * i:16 * i + 16] = 0
    q = queries(n, 24, dtype, 42)[:, 8:16]
    got = q3.attention_prompt(*p.handles([0, n]), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    check_attention(got, q, k, v, range(1, n + 1), dtype, H if dtype == BF16 else 0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_caches_at_16_bytes(q3, dtype):
    """Pages that begin 16 bytes behind a 32-byte boundary, which is all that is asked for."""
    n, off16 = 150, 16 // torch.empty((), dtype=dtype).element_size()
    p = Paged([n], 2, 16, dtype, seed=70).fill(71)
    for name in ("k", "v"):
        x = getattr(p, name)
        buf = torch.full((x.numel() + off16,), NAN, dtype=dtype, device="cuda")
        moved = buf[off16:].view(x.shape)
        assert buf.data_ptr() % 32 == 0 and moved.data_ptr() % 32 == 16
        moved.copy_(x)
        setattr(p, name, moved)
    q = queries(n, 8, dtype, 72)
    check_attention(q3.attention_prompt(*p.handles([0, n]), q), q, *p.rows(0), range(1, n + 1), dtype,
                    H if dtype == BF16 else 0.0)
    check_attention(q3.attention_paged(*p.handles(), q[-1:]), q[-1:], *p.rows(0), [n], dtype)
    x, w, at = queries(n, 8, dtype, 73), torch.ones(128, device="cuda"), torch.arange(n, device="cuda")
    k, v = x[:, 4:6], x[:, 6:]
    got = q3.kv_append(*p.handles([0, n]), x[:, :4], k, v, w, w)
    check_rotated(got, x[:, :4], w, at, dtype)
    check_rotated(p.rows(0)[0].to(dtype), k, w, at, dtype)
    assert torch.equal(p.rows(0)[1], v.double())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_prompt_infinities(q3, dtype):
    """An infinite key element makes a score -inf (weight 0) or +inf (a row of NaN), an infinite value one column."""
    n = 130
    p = Paged([n], 2, 16, dtype, seed=74).fill(75)
    q = queries(n, 4, dtype, 76)
    page, slot = p.where(0, [70])
    p.k[page, 0, slot, 5] = math.inf
    p.v[page, 1, slot, 9] = math.inf
    got, (k, v) = q3.attention_prompt(*p.handles([0, n]), q).double(), p.rows(0)
    rounding = H if dtype == BF16 else 0.0
    up = (q[:, :2, 5] > 0) & (torch.arange(n, device="cuda") >= 70)[:, None]
    assert up.any() and (~up).any() and got[:, :2][up].isnan().all()
    for h in range(2):
        keep = (~up[:, h]).nonzero()[:, 0]
        check_attention(got[keep, h:h + 1], q[keep, h:h + 1], k[:, :1], v[:, :1], keep + 1, dtype, rounding)
    assert (got[70:, 2:, 9] == math.inf).all()
    v[70, 1, 9] = 0.0
    got[70:, 2:, 9] = attend(q[70:, 2:].double(), k[:, 1:], v[:, 1:], range(71, n + 1))[0][:, :, 9]
    check_attention(got[:, 2:], q[:, 2:], k[:, 1:], v[:, 1:], range(1, n + 1), dtype, rounding)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [
    (32, 8, 16, [16], [1000]), (16, 1, 64, [100], [3001]), (8, 2, 16, [70, 3, 0, 5], [900, 2000, 40, 5]),
    (4, 4, 32, [500], [500]), (5, 1, 256, [37, 1], [2600, 4097]), (12, 4, 16, [33], [513]), (2, 2, 128, [1], [6000]),
    (16, 8, 16, [40, 30], [20, 1100]), (32, 8, 16, [65], [2111]), (8, 8, 16, [3, 3], [1500, 700]),
])
def test_attention_prompt_few_rows_many_keys(q3, dtype, heads, n_kv, page, rows, lens):
    """Few items, whose keys several multiprocessors share."""
    p = Paged(lens, n_kv, page, dtype, seed=80).fill(81)
    q = queries(sum(rows), heads, dtype, 82)
    off = offsets(rows)
    out = torch.full(q.shape, 3.0, dtype=dtype, device="cuda")
    q3.attention_prompt(*p.handles(off), q, out=out)
    for s, n in enumerate(lens):
        a, b = off[s], off[s + 1]
        seen = [max(0, n - rows[s] + i + 1) for i in range(rows[s])]
        check_attention(out[a:b], q[a:b], *p.rows(s), seen, dtype, H if dtype == BF16 else 0.0)
    again = q3.attention_prompt(*p.handles(off), q)
    assert torch.equal(again, out) and q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_prompt_few_rows_bad_pages_and_nan(q3, dtype):
    """Of keys that several multiprocessors share: a page outside the cache reads as zeros, a NaN at a hidden position
    stays hidden and one that is seen shows in its rows."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX
    n, rows = 2000, 20
    p = Paged([n], 2, 16, dtype, seed=83).fill(84)
    k, v = p.rows(0)
    for i, bad in ((3, -1), (60, 1 << 29), (120, p.n_pages)):
        p.table[0, i] = bad
        k[16 * i:16 * i + 16] = 0
        v[16 * i:16 * i + 16] = 0
    page, slot = p.where(0, [n - 8])
    p.k[page, 0, slot, 7] = NAN
    p.v[page, 1, slot, 3] = NAN
    q = queries(rows, 8, dtype, 85)
    got = q3.attention_prompt(*p.handles([0, rows]), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    seen = torch.arange(n - rows + 1, n + 1)
    before = rows - 8                                        # rows that end before position n - 8
    check_attention(got[:before], q[:before], k, v, seen[:before], dtype, H if dtype == BF16 else 0.0)
    assert got[before:, :4].isnan().all() and got[before:, 4:, 3].isnan().all()
    got[before:, 4:, 3] = 0.0
    assert not got[before:, 4:].isnan().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_few_rows_replayed(q3, dtype):
    """A captured call is replayed while the sequences grow from a few keys, which one multiprocessor takes, to many."""
    p = Paged([3000, 1200], 2, 16, dtype, seed=86).fill(87)
    cache, batch = p.handles([0, 9, 14])
    q = queries(14, 8, dtype, 88)
    out = torch.zeros_like(q)
    q3.attention_prompt(cache, batch, q, out=out)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        q3.attention_prompt(cache, batch, q, out=out)
    for lens in ((9, 5), (300, 1200), (3000, 40), (1030, 520), (0, 3)):
        p.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for s, (a, b) in enumerate(((0, 9), (9, 14))):
            k, v = p.rows(s)
            seen = [max(0, lens[s] - (b - a) + i + 1) for i in range(b - a)]
            check_attention(out[a:b], q[a:b], k[:lens[s]], v[:lens[s]], seen, dtype, H if dtype == BF16 else 0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_on_two_streams(q3, dtype):
    """Clusters of two calls wait for multiprocessors beside each other, and each call's result is as alone."""
    sets = []
    for seed, rows, lens in ((90, [20, 3], [1900, 800]), (93, [40], [2500])):
        p = Paged(lens, 8, 16, dtype, seed=seed).fill(seed + 1)
        q = queries(sum(rows), 16, dtype, seed + 2)
        cache, batch = p.handles(offsets(rows))
        sets.append((p, cache, batch, q, q3.attention_prompt(cache, batch, q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(12):
        for i, (_, cache, batch, q, _, stream) in enumerate(sets):
            with torch.cuda.stream(stream):
                outs[i].append(q3.attention_prompt(cache, batch, q))
    torch.cuda.synchronize()
    for got, (_, _, _, _, alone, _) in zip(outs, sets):
        assert all(torch.equal(g, alone) for g in got)


def test_offsets_that_do_not_rise(q3):
    """Broken row offsets touch nothing outside the rows and fault nothing."""
    p = Paged([50, 50, 50], 2, 16, BF16, seed=43).fill(44)
    q = queries(20, 4, BF16, 45)
    out = torch.full((20, 4, 128), 7.0, dtype=BF16, device="cuda")
    k = queries(20, 2, BF16, 46)
    for off in ([5, 3, -4, 1000], [20, 10, 5, 0], [-100, 100, 200, 300], [0, 1 << 30, -(1 << 30), 20]):
        cache, batch = p.handles(off)
        q3.kv_append(cache, batch, q, k, k)
        q3.attention_prompt(cache, batch, q, out=out)
    q3.device_status()


# ---- as a server uses them -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompts_in_chunks_then_decoding(q3, dtype):
    """Two prompts appended and attended in chunks, then decoding steps: each row's result is the attention over all
    rotated keys so far."""
    heads, n_kv, page, eps_p = 8, 2, 16, (H if dtype == BF16 else 0.0)
    final = [75, 140]
    p = Paged(final, n_kv, page, dtype, seed=50)
    p.kv_len.zero_()
    g = torch.Generator(device="cuda").manual_seed(51)
    qkv = [torch.randn((n, heads + 2 * n_kv, 128), generator=g, device="cuda") for n in final]
    qn, kn = (1 + 0.2 * torch.randn(128, generator=g, device="cuda") for _ in range(2))
    done = [0, 0]
    steps = [(40, 100), (30, 0), (0, 33)] + [(1, 1)] * 5
    work = None
    for rows in steps:
        off = offsets(rows)
        x = torch.cat([qkv[s][done[s]:done[s] + rows[s]] for s in range(2)])
        for s in range(2):
            done[s] += rows[s]
        p.kv_len.copy_(torch.tensor(done, dtype=torch.int32))
        cache, batch = p.handles(off)
        q = q3.kv_append(cache, batch, x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:], qn, kn)
        if rows == (1, 1):
            work = q3.attention_paged_workspace(cache, heads) if work is None else work
            got = q3.attention_paged(cache, batch, q, work=work)
        else:
            got = q3.attention_prompt(cache, batch, q)
        for s in range(2):
            if rows[s] == 0:
                continue
            k, v = (t[:done[s]] for t in p.rows(s))
            pos = torch.arange(done[s], device="cuda")
            check_rotated(k, qkv[s][:done[s], heads:heads + n_kv], kn, pos, dtype)
            assert torch.equal(v, qkv[s][:done[s], heads + n_kv:].to(dtype).double())
            mine = slice(off[s], off[s + 1])
            check_rotated(q[mine], x[mine, :heads], qn, pos[-rows[s]:], dtype)
            check_attention(got[mine], q[mine], k, v, range(done[s] - rows[s] + 1, done[s] + 1), dtype, eps_p)
    assert done == [sum(r[s] for r in steps) for s in range(2)] and q3.device_status() == 0


def test_captured_step_replayed(q3):
    """One decoding step as a graph, replayed as the sequences grow: lengths and pages are read at each replay."""
    heads, n_kv = 16, 8
    p = Paged([200, 333], n_kv, 64, BF16, seed=60).fill(61)
    lens = torch.tensor([190, 0], dtype=torch.int32)
    x = queries(2, heads + 2 * n_kv, F32, 62)
    cache, batch = p.handles([0, 1, 2])
    out, rq = (torch.empty((2, heads, 128), dtype=BF16, device="cuda") for _ in range(2))
    work = q3.attention_paged_workspace(cache, heads)

    def step():
        q3.kv_append(cache, batch, x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:], q_out=rq)
        q3.attention_paged(cache, batch, rq, out=out, work=work)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        lens += torch.tensor([2, 83 * (i > 0)], dtype=torch.int32)
        p.kv_len.copy_(lens)
        x.copy_(queries(2, heads + 2 * n_kv, F32, 63 + i))
        graph.replay()
        for s in range(2):
            k, v = p.rows(s)
            n = int(lens[s])
            check_attention(out[s:s + 1], rq[s:s + 1], k[:n], v[:n], [n], BF16)
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_prompts_replayed(q3, dtype):
    """A captured append and prompt attention, replayed with other offsets and lengths, more items than the GPU has SMs."""
    rows_max, heads, n_kv = 1500, 16, 8
    p = Paged([900, 1100, 700], n_kv, 16, dtype, seed=64).fill(65)
    off = torch.tensor([0, 300, 900, 1400], dtype=torch.int32, device="cuda")
    x = queries(rows_max, heads + 2 * n_kv, F32, 66)
    from metalqwen3_b200.q3cu import KVBatch
    cache, batch = p.handles()[0], KVBatch(p.kv_len, p.table, off)
    rq, out = (torch.full((rows_max, heads, 128), 5.0, dtype=dtype, device="cuda") for _ in range(2))

    def step():
        q3.kv_append(cache, batch, x[:, :heads], x[:, heads:heads + n_kv], x[:, heads + n_kv:], q_out=rq)
        q3.attention_prompt(cache, batch, rq, out=out)

    p.kv_len.copy_(torch.tensor([300, 600, 500], dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rows, lens in (((300, 600, 500), (300, 600, 500)), ((1, 1100, 399), (1, 1100, 700)), ((0, 0, 64), (0, 900, 64)),
                       ((800, 33, 600), (900, 1033, 650))):
        off.copy_(torch.tensor(offsets(rows), dtype=torch.int32))
        p.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        first = 0
        for s, (r, n) in enumerate(zip(rows, lens)):
            if r:
                k, v = (t[:n] for t in p.rows(s))
                pick = sorted({0, 1 % r, r // 3, r // 2, r - 1})           # the others are the same code
                at = torch.tensor([first + i for i in pick], device="cuda")
                check_attention(out[at], rq[at], k, v, [n - r + 1 + i for i in pick], dtype, H if dtype == BF16 else 0.0)
                assert torch.isfinite(out[first:first + r]).all()
            first += r
        assert (out[first:] == 5.0).all()
    assert q3.device_status() == 0


def test_calls_on_a_given_stream(q3):
    """`stream` in place of the current one, with the binding's own outputs and workspace."""
    p = Paged([70, 1200], 2, 16, BF16, seed=67).fill(68)
    q, k = queries(2, 8, BF16, 69), queries(2, 2, BF16, 70)
    cache, batch = p.handles([0, 1, 2])
    want = q3.attention_paged(cache, batch, q), q3.attention_prompt(cache, batch, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(10):
        got = q3.attention_paged(cache, batch, q, stream=side), q3.attention_prompt(cache, batch, q, stream=side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    rq = q3.kv_append(cache, batch, q, k, k, stream=side)
    side.synchronize()
    check_rotated(rq, q, None, torch.tensor([69, 1199], device="cuda"), BF16)
    assert q3.device_status(side) == 0


def test_two_streams_at_once(q3):
    """Calls on two streams with a workspace each, many times: every result equals the call alone."""
    sets = []
    for i in range(2):
        p = Paged([3000 + 500 * i, 41, 900], 8, 16, BF16, seed=70 + i).fill(72 + i)
        q = queries(3, 32, BF16, 74 + i)
        cache, batch = p.handles([0, 1, 2, 3])
        sets.append((torch.cuda.Stream(), p, cache, batch, q, q3.attention_paged_workspace(cache, 32),
                     q3.attention_paged(cache, batch, q), q3.attention_prompt(cache, batch, q)))
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        for stream, p, cache, batch, q, work, one, prompt in sets:
            with torch.cuda.stream(stream):
                results.append((q3.attention_paged(cache, batch, q, work=work), one))
                results.append((q3.attention_prompt(cache, batch, q), prompt))
    torch.cuda.synchronize()
    for got, alone in results:
        assert torch.equal(got, alone)
    assert q3.device_status() == 0


# ---- refusals ------------------------------------------------------------------------------------

def test_refusals(q3):
    from metalqwen3_b200.q3cu import KVBatch, KVCache, Q3Error
    p = Paged([20, 20], 2, 16, BF16, seed=80).fill(81)
    cache, batch = p.handles([0, 1, 2])
    q, k = queries(2, 4, BF16, 82), queries(2, 2, BF16, 83)

    def refused(status, call):
        with pytest.raises(Q3Error) as e:
            call()
        assert e.value.status == status

    refused(1, lambda: q3.attention_prompt(cache, batch, q.float()))                       # types differ
    refused(1, lambda: q3.attention_paged(cache, batch, queries(2, 3, BF16, 84)))          # heads % n_kv
    refused(1, lambda: q3.attention_paged(cache, batch, queries(2, 34, BF16, 84)))         # 17 to a kv head
    refused(1, lambda: q3.attention_paged(cache, batch, q, work=torch.empty(0, dtype=torch.uint8, device="cuda")))
    refused(1, lambda: q3.attention_paged(cache, batch, q, out=q))
    refused(1, lambda: q3.attention_prompt(cache, batch, q, out=q))
    refused(1, lambda: q3.attention_prompt(cache, p.handles()[1], q))                      # no row offsets
    refused(1, lambda: q3.kv_append(cache, batch, q, k, k, theta=0.0))
    refused(2, lambda: q3.attention_paged(cache, batch, torch.empty(2 * 4 * 128 + 8, dtype=BF16, device="cuda")
                                          [4:4 + 1024].view(2, 4, 128)))
    odd = torch.zeros((4, 2, 24, 128), dtype=BF16, device="cuda")
    refused(1, lambda: q3.attention_paged(KVCache(odd, odd), batch, q))                    # page of 24
    short = torch.zeros((4, 2, 16, 64), dtype=BF16, device="cuda")
    refused(1, lambda: q3.attention_paged(KVCache(short, short), batch, q))                # head_dim 64
    for bad in (lambda: KVCache(p.k, p.v.float()), lambda: KVCache(p.k[:, :, ::2], p.v[:, :, ::2]),
                lambda: KVBatch(p.kv_len, p.table[:1]), lambda: q3.attention_paged(cache, batch, q[:1]),
                lambda: q3.kv_append(cache, batch, q, k, k[:1]),
                lambda: q3.attention_paged(cache, batch, q, out=torch.empty((2, 4, 64), dtype=BF16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: KVBatch(p.kv_len.long(), p.table), lambda: KVCache(p.k.half(), p.v.half()),
                lambda: q3.attention_paged(cache, batch, q, out=torch.empty((2, 4, 128), device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    assert q3.device_status() == 0


def test_empty_batches(q3):
    """No sequences, no rows: nothing is launched and nothing written."""
    from metalqwen3_b200.q3cu import KVBatch
    p = Paged([20], 2, 16, BF16, seed=85).fill(86)
    cache, batch = p.handles([0, 0])
    none = KVBatch(p.kv_len[:0], p.table[:0], torch.zeros(1, dtype=torch.int32, device="cuda"))
    q, k = queries(0, 4, BF16, 87), queries(0, 2, BF16, 88)
    assert q3.attention_prompt(cache, batch, q).shape == (0, 4, 128)
    assert q3.attention_paged(cache, none, q).shape == (0, 4, 128)
    q3.kv_append(cache, batch, q, k, k)
    out = torch.full((3, 4, 128), 7.0, dtype=BF16, device="cuda")
    q3.attention_prompt(cache, none, queries(3, 4, BF16, 89), out=out)
    q3.attention_prompt(cache, batch, queries(3, 4, BF16, 89), out=out)
    assert (out == 7.0).all() and q3.device_status() == 0
