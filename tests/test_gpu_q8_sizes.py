"""Prompts and shared positions over a Q8_0 cache whose values and keys differ widely in size, against the formula in
binary64.  Tolerances as in test_gpu_paged_q8.py, with the elements rounded as the products take them (11 bits of a scale,
11 of the product; here of each by itself, as the tiles' lifts are powers of two).  The floor of a probability is 2^-32, and
2^-24 where a position before holds larger values (by no more than 2^8 more is O kept than the values at hand need), but
never relative to values that carry no weight: their part of a result is bounded by itself.
"""
import math

import pytest
import torch

from test_gpu_kv_forms import Quantised
from test_gpu_paged import BF16, F32, H, U, attend, queries
from test_gpu_paged_q8 import check_attention

pytestmark = pytest.mark.gpu
W = 2.0 ** -11


def bits11(x):
    """x (f64) rounded to 11 bits, whatever its size."""
    m, e = torch.frexp(x)
    return torch.ldexp(m.half().double(), e)


def rounded(p, s):
    """Keys and values of sequence s as the products take them."""
    page, slot = p.where(s, range(max(p.lens[s], 0)))
    return tuple(bits11(bits11(c[page, :, slot].double()).repeat_interleave(64, -1) * t[page, :, slot].double())
                 for t, c in ((p.k, p.ks), (p.v, p.vs)))


def check(got, q, k, v, seen, light=()):
    """`light`: positions whose values are large and carry no weight."""
    o, pv, a = attend(q.double(), k, v, seen)
    keep = torch.ones(k.shape[0], dtype=torch.bool, device=k.device)
    keep[list(light)] = False
    only = v.clone()
    only[keep] = 0
    top = float(v[keep].abs().max())
    ds = 160 * U * a + math.sqrt(128) * 2.0 ** -39 * float(q.abs().max()) * float(k.abs().max())
    tol = (torch.expm1(2 * ds) + (k.shape[0] + 64) * U + W) * pv + attend(q.double(), k, only, seen)[1]
    tol = tol + k.shape[0] * (2.0 ** -24 + 2.0 ** -39) * 1.01 * top
    tol = tol + H * (o.abs() + tol)
    bad = ~((got.double() - o).abs() <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - o).abs().max()), float(tol.max()))


def light_tiles(lens, n_kv, at, key, size, seed):
    """Sequences whose positions `at` hold values `size` times larger, and keys whose first element is `key` (elsewhere 0):
    with queries whose first element is 40, their scores are lower by 40 key / sqrt(128)."""
    p = Quantised(lens, n_kv, 16, seed=seed).fill(seed + 1)
    for s, n in enumerate(lens):
        page, slot = p.where(s, range(n))
        p.k[page, :, slot, 0] = 0
        page, slot = page[at], slot[at]
        p.vs[page, :, slot] *= size
        p.k[page, :, slot, :64] = 0
        p.k[page, :, slot, 0] = -127
        p.ks[page, :, slot, 0] = key / 127
    return p


def light_queries(rows, heads, seed):
    q = queries(rows, heads, BF16, seed, 1.0)
    q[..., 0] = 40.0
    return q


@pytest.mark.parametrize("key", [12.0, 30.0])           # weights of 2^-60 and of less than 2^-126
@pytest.mark.parametrize("size", [2.0 ** 28, 2.0 ** 36])
@pytest.mark.parametrize("first", [0, 128, 256])
@pytest.mark.parametrize("rows", [600, 70, 5])
def test_large_values_without_weight(q3, key, size, first, rows):
    """Prompts, a chunk, a few rows: what carries the weight keeps its bits, whatever lies before it."""
    n = 600
    at = list(range(first, first + 128))
    p = light_tiles([n], 2, at, key, size, 70)
    q = light_queries(rows, 8, 72)
    got = q3.attention_prompt(*p.handles([0, rows]), q)
    assert q3.device_status() == 0
    k, v = rounded(p, 0)
    # (from the first row whose weight is elsewhere, among at least eight positions)
    start = max(0, (136 if first == 0 else 0) - (n - rows))
    check(got[start:], q[start:], k, v, range(n - rows + 1 + start, n + 1), at)


@pytest.mark.parametrize("key", [12.0, 30.0])
@pytest.mark.parametrize("size", [2.0 ** 28, 2.0 ** 36])
def test_large_values_without_weight_shared(q3, key, size):
    from metalqwen3_b200.q3cu import KVPrefix
    n, at = 3000, list(range(128, 384))
    p = light_tiles([n] * 5, 2, at, key, size, 74)
    p.table[1:, :n // 16] = p.table[0, :n // 16]        # shared up to a page's end: 2,992
    i32 = dict(dtype=torch.int32, device="cuda")
    q = light_queries(5, 8, 76)
    cache, batch = p.handles()
    got = q3.attention_shared(cache, batch, KVPrefix(torch.tensor([0, 5], **i32), torch.tensor([2992], **i32)), q)
    assert q3.device_status() == 0
    for s in range(5):
        check(got[s:s + 1], q[s:s + 1], *rounded(p, s), [n], at)


@pytest.mark.parametrize("n", [400, 2960])
@pytest.mark.parametrize("rows", [384, 70, 9])
def test_larger_values_behind_change_nothing(q3, rows, n):
    """Positions that a row does not see, in a later tile, 2^140 times larger: the row's bits stay."""
    got = []
    for size in (1.0, 2.0 ** 70):
        p = Quantised([n], 2, 16, seed=77).fill(78, 2.0 ** -60)
        page, slot = p.where(0, range(n - n % 128, n))
        for _ in range(2):                              # (2^140 is no binary32)
            p.vs[page, :, slot] *= size
        if rows == 9:                                   # all but the last row in the tile before
            p.kv_len[0] = n - n % 128 + 4
        got.append(q3.attention_prompt(*p.handles([0, rows]), queries(rows, 8, BF16, 79)))
    early = rows - (4 if rows == 9 else 16)
    assert early > 0 and torch.equal(got[0][:early], got[1][:early]) and (got[0][:early] != 0).any()
    assert torch.isfinite(got[1].float()).all() and q3.device_status() == 0


@pytest.mark.parametrize("rows,n", [(300, 300), (100, 700), (7, 3000)])
def test_small_scales_cost_no_second_computation(q3, rows, n):
    """A value group and a key group 2^-60 as large as the others, in the tile that the last rows see in part: what the
    products give of them is 0 (f16 has no less than 2^-24, the largest are lifted to 2^15), so the results are, bit for bit,
    those of scales that are 0, which no row is computed again for."""
    got = []
    for size in (0.0, 2.0 ** -60):
        p = Quantised([n], 2, 16, seed=80).fill(81)
        page, slot = p.where(0, [n - rows // 2 - 1, n - rows])
        p.vs[page, 0, slot, 1] *= size
        p.ks[page, 1, slot, 0] *= size
        got.append(q3.attention_prompt(*p.handles([0, rows]), queries(rows, 8, BF16, 82)))
    assert torch.equal(got[0], got[1]) and q3.device_status() == 0


def test_time_for_second_computations_runs_out(q3):
    """The last position's values 2^40 times larger, behind 300,000: the rows before it are computed again for a second, and
    what is left keeps the tensor cores' result."""
    from metalqwen3_b200.q3cu import DEV_TIMEOUT
    n, rows = 300_000, 1280
    p = Quantised([n], 8, 256, seed=83).fill(84)
    page, slot = p.where(0, [n - 1])
    p.vs[page, 0, slot] *= 2.0 ** 40
    got = q3.attention_prompt(*p.handles([0, rows]), queries(rows, 32, BF16, 85))
    try:
        timed_out = q3.device_status() == DEV_TIMEOUT
    except Exception:
        timed_out = True
    assert timed_out and torch.isfinite(got.float()).all()
    assert q3.device_status() == 0


@pytest.mark.parametrize("io", [F32, BF16])
@pytest.mark.parametrize("size_q,size_kv", [(1e-33, 1e33), (1e-36, 1e36), (1e33, 1e-33), (1e-30, 1e30)])
def test_one_token_far_from_1(q3, io, size_q, size_kv):
    """Keys and values up to the end of binary32 with scores as usual, alone and behind a shared prefix."""
    from metalqwen3_b200.q3cu import KVPrefix
    for heads in (8, 32):
        p = Quantised([300, 300], 2, 16, seed=86).fill(87, size_kv)
        p.table[1, :16] = p.table[0, :16]
        q = queries(2, heads, io, 88, size_q)
        got = [q3.attention_paged(*p.handles(), q)]
        if io == BF16:
            i32 = dict(dtype=torch.int32, device="cuda")
            got.append(q3.attention_shared(*p.handles(), KVPrefix(torch.tensor([0, 2], **i32), torch.tensor([256], **i32)), q))
        for x, elements in zip(got, (p.rows, lambda s: tuple(torch.cat([a[:256], b[256:]]) for a, b in zip(rounded(p, s), p.rows(s))))):
            for s in range(2):
                k, v = elements(s)
                check_attention(x[s:s + 1], q[s:s + 1], k, v, [300], io, W if io == BF16 else 0.0, 2.0 ** -32 if len(got) > 1 else 2.0 ** -39)
    assert q3.device_status() == 0


@pytest.mark.parametrize("n,rows", [(300, 300), (300, 60), (2000, 1800), (2000, 90)])
def test_sizes_from_end_to_end(q3, n, rows):
    """Values 2^130 times larger, in one case behind zeros in the tile that a row sees in part, in the other seen but without
    weight: what is lowered for them does not go under."""
    big = n // 128 * 128
    for light in (False, True):
        p = Quantised([n], 2, 16, seed=95).fill(96, 2.0 ** -60)
        page, slot = p.where(0, range(n))
        p.k[page, :, slot, 0] = 0
        at = list(range(big, big + 1)) if light else list(range(big + 1, n))
        if not light:
            p.vs[page[big], :, slot[big]] = 0
        for _ in range(2):
            p.vs[page[at], :, slot[at]] *= 2.0 ** 65
        p.ks[page, :, slot] *= 2.0 ** 60
        if light:
            p.k[page[at], :, slot[at], :64] = 0
            p.k[page[at], :, slot[at], 0] = -127
            p.ks[page[at], :, slot[at], 0] = 60.0 / 127
        q = light_queries(rows, 8, 98)
        got = q3.attention_prompt(*p.handles([0, rows]), q)
        k, v = rounded(p, 0)
        pick = [i for i in range(rows) if (i >= rows - n + big) == light][:: 1 + rows // 64]
        if not light:
            pick.append(rows - n + big)                 # (the one that sees the zeros)
        check(got[pick], q[pick], k[:big + 1] if not light else k, v[:big + 1] if not light else v,
              [n - rows + i + 1 for i in pick], at if light else ())
    assert q3.device_status() == 0
