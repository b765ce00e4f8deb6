"""The paged-cache operators where one element, one order or one stream decides.  Formulas, tolerances and helpers are
those of test_gpu_paged.py."""
import math
import os
import subprocess

import pytest
import torch

from test_gpu_paged import BF16, F32, H, NAN, Paged, attend, check_attention, offsets, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [list(range(1, 33)), [0] * 32, [1] * 32, [32, 0] * 16])
def test_nothing_to_join_then_dependent_kernels(q3, dtype, lens):
    """One-token attention of sequences no longer than a tile, which no two multiprocessors share, between kernels that
    start as early as they may: one that reads its result and one that overwrites its queries."""
    p, heads, steps = Paged(lens, 2, 16, dtype, seed=110).fill(111), 8, 200
    cache, batch = p.handles(list(range(33)))
    other = Paged([64] * 32, 2, 16, dtype, seed=112, fill=0.0).handles()[0]      # what the steps append to
    x = torch.stack([queries(32, heads, dtype, 200 + i) for i in range(8)])
    k = queries(32, 2, dtype, 113)
    work = q3.attention_paged_workspace(cache, heads)
    q = torch.empty_like(x[0])
    outs, turned = (torch.empty((steps,) + x[0].shape, dtype=dtype, device="cuda") for _ in range(2))

    def step(i, out, turn, wait=lambda: None):
        q3.kv_append(other, batch, x[i % 8], k, k, q_out=q)
        wait()
        q3.attention_paged(cache, batch, q, out=out, work=work)
        wait()
        q3.kv_append(other, batch, out, k, k, q_out=turn)
        wait()

    alone = torch.empty((8, 2) + x[0].shape, dtype=dtype, device="cuda")
    for i in range(8):
        step(i, alone[i, 0], alone[i, 1], torch.cuda.synchronize)
        step(i, alone[i, 0], alone[i, 1], torch.cuda.synchronize)
    for s, n in enumerate(lens):                             # q holds the last step's rotated queries
        check_attention(alone[7, 0, s:s + 1], q[s:s + 1], *p.rows(s), [n], dtype)
    graph = torch.cuda.CUDAGraph()
    for captured in (False, True):
        if captured:
            outs.fill_(3), turned.fill_(3)
            with torch.cuda.graph(graph):
                for i in range(steps):
                    step(i, outs[i], turned[i])
            graph.replay()
        else:
            for i in range(steps):
                step(i, outs[i], turned[i])
        torch.cuda.synchronize()
        for i in range(steps):
            live = torch.tensor(lens, device="cuda") > 0     # padding rows are not turned
            assert torch.equal(outs[i], alone[i % 8, 0]) and torch.equal(turned[i][live], alone[i % 8, 1][live])
    assert q3.device_status() == 0


def test_current_and_given_stream_at_once(q3):
    """Calls on the current stream and, with nothing between them, on a given one: the memory that they make for
    themselves is apart, and each result is as alone."""
    sets = []
    for i in range(2):
        p = Paged([30000, 7000], 2, 16, BF16, seed=120 + i).fill(122 + i)
        q = queries(2, 32, BF16, 124 + i)
        cache, batch = p.handles([0, 1, 2])
        rows = queries(2, 36, BF16, 126 + i)
        sets.append((p, cache, batch, q, rows))

    def calls(i, stream=None):
        _, cache, batch, q, rows = sets[i]
        one = q3.attention_paged(cache, batch, q, stream=stream)
        prompt = q3.attention_prompt(cache, batch, q, stream=stream)
        return one, prompt, q3.kv_append(other, batch, rows[:, :32], rows[:, 32:34], rows[:, 34:], stream=stream)

    p = sets[0][0]                                           # appended to, and read by nothing
    other = type(sets[0][1])(torch.zeros_like(p.k), torch.zeros_like(p.v))
    alone = []
    for i in range(2):
        alone.append(calls(i))
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    freed = torch.empty((2, 32, 128), dtype=BF16, device="cuda")
    at = freed.data_ptr()
    del freed
    assert all(t.data_ptr() != at for t in calls(1, side))
    got = []
    for _ in range(50):
        got.append((0, calls(0)))
        got.append((1, calls(1, side)))
    torch.cuda.synchronize()
    for i, results in got:
        assert all(torch.equal(a, b) for a, b in zip(results, alone[i]))
    assert q3.device_status() == 0 and q3.device_status(side) == 0


def rounding(dtype):
    return H if dtype == BF16 else 0.0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", [math.inf, -math.inf, NAN, 3e38, -3e38])
@pytest.mark.parametrize("n,rows,at", [(300, 300, 200), (600, 600, 290), (2000, 20, 1986)])
def test_hidden_values_reach_no_earlier_row(q3, dtype, what, n, rows, at):
    """A value in one column of one position, at each of eight positions running: rows before it are as if it was not
    there, in whole items and in those that several multiprocessors share."""
    p = Paged([n], 2, 16, dtype, seed=100).fill(101)
    page, slot = p.where(0, range(n))
    q = queries(rows, 8, dtype, 102)
    clean = p.v.clone()
    for hidden in range(at, at + 8):
        p.v.copy_(clean)
        p.v[page[hidden], :, slot[hidden], 17 * (hidden - at)] = what
        got = q3.attention_prompt(*p.handles([0, rows]), q)
        k, v = p.rows(0)
        before = hidden - (n - rows)
        check_attention(got[:before], q[:before], k[:hidden], v[:hidden], range(n - rows + 1, hidden + 1), dtype,
                        rounding(dtype))
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,rows,at", [(150, 150, 0), (150, 150, 1), (150, 150, 63), (150, 150, 64), (300, 300, 127),
                                       (300, 300, 128), (1500, 10, 0), (1500, 10, 1486)])
def test_infinite_keys_and_values(q3, dtype, n, rows, at):
    """An infinite element of a key, wherever the key lies, makes its score -inf (weight 0: the other keys share the row)
    or +inf (a row of NaN); an infinite value makes its column infinite."""
    p = Paged([n], 2, 16, dtype, seed=103).fill(104)
    page, slot = p.where(0, [at])
    p.k[page, 0, slot, 5] = math.inf
    p.v[page, 1, slot, 9] = math.inf
    q = queries(rows, 4, dtype, 105)
    got, (k, v) = q3.attention_prompt(*p.handles([0, rows]), q).double(), p.rows(0)
    position = torch.arange(n - rows, n, device="cuda")
    sees = position >= at
    up = (q[:, :2, 5] > 0) & sees[:, None]
    assert up.any() and (sees[:, None] & ~up).any() and got[:, :2][up].isnan().all()
    for h in range(2):
        keep = (~up[:, h] & (position > 0)).nonzero()[:, 0]       # row 0 has no other key
        check_attention(got[keep, h:h + 1], q[keep, h:h + 1], k[:, :1], v[:, :1], position[keep] + 1, dtype,
                        rounding(dtype))
    assert (got[sees, 2:, 9] == math.inf).all()
    v[at, 1, 9] = 0.0
    got[sees, 2:, 9] = attend(q[sees][:, 2:].double(), k[:, 1:], v[:, 1:], position[sees] + 1)[0][:, :, 9]
    check_attention(got[:, 2:], q[:, 2:], k[:, 1:], v[:, 1:], position + 1, dtype, rounding(dtype))
    assert q3.device_status() == 0


@pytest.mark.parametrize("io,cache_t", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("n,at", [(1, 0), (40, 0), (40, 39), (3000, 0), (3000, 1777), (3000, 2999)])
def test_one_token_infinities_are_right_or_nan(q3, io, cache_t, n, at):
    """An infinite key's heads and an infinite value's column are as the formula has them or NaN, the others as ever."""
    p = Paged([n], 2, 16, cache_t, seed=106).fill(107)
    page, slot = p.where(0, [at])
    p.k[page, 0, slot, 5] = math.inf
    p.v[page, 1, slot, 9] = math.inf
    q = queries(1, 4, io, 108)
    got, (k, v) = q3.attention_paged(*p.handles(), q).double(), p.rows(0)
    for h in range(2):                                       # a score of +inf, or -inf and no other: NaN
        if not got[:, h].isnan().all():
            assert n > 1 and q[0, h, 5] < 0
            check_attention(got[:, h:h + 1], q[:, h:h + 1], k[:, :1], v[:, :1], [n], io)
    assert ((got[:, 2:, 9] == math.inf) | got[:, 2:, 9].isnan()).all()
    v[at, 1, 9] = 0.0
    got[:, 2:, 9] = attend(q[:, 2:].double(), k[:, 1:], v[:, 1:], [n])[0][:, :, 9]
    check_attention(got[:, 2:], q[:, 2:], k[:, 1:], v[:, 1:], [n], io)
    assert q3.device_status() == 0


def test_prompt_items_in_any_order(tmp_path):
    """Every item of a launch is found at its index, whatever order the indices come in (check_prompt_order.cu)."""
    from metalqwen3_b200.build import CSRC
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "check_prompt_order")
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--fmad=false", "-I", CSRC, "-I",
                    os.path.join(root, "include"), os.path.join(root, "tests", "native", "check_prompt_order.cu"), "-o", exe],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,rows", [(4096, 4096), (20000, 24)])
def test_a_nan_is_not_looked_for_in_every_row(q3, dtype, n, rows):
    """A NaN that all rows see, in a key or in one column of a value: NaN where the formula has it, every other column
    right, and in a long prompt no row-by-row computation, which would take some hundred times the call's usual time."""
    p = Paged([n], 2, 64, dtype, seed=130).fill(131)
    q = queries(rows, 8, dtype, 132)
    handles, out = p.handles([0, rows]), torch.empty_like(q)
    page, slot = p.where(0, [0])
    pick = torch.tensor(sorted({0, 1, rows // 3, rows - 2, rows - 1}), device="cuda")
    seen = pick + (n - rows + 1)

    def call():
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        q3.attention_prompt(*handles, q, out=out)
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    call()
    usual = min(call() for _ in range(5))
    p.v[page, :, slot, 3] = NAN
    assert min(call() for _ in range(3)) < 60 * usual or rows < n
    assert out[:, :, 3].isnan().all() and not out[:, :, 4:].isnan().any()
    k, v = p.rows(0)
    v[0, :, 3] = 0.0
    got = out[pick].double()
    got[:, :, 3] = attend(q[pick].double(), k, v, seen)[0][:, :, 3]
    check_attention(got, q[pick], k, v, seen, dtype, rounding(dtype))
    p.k[page, 0, slot, 7] = NAN
    assert min(call() for _ in range(3)) < 60 * usual or rows < n
    assert out[:, :4].isnan().all() and not out[:, 4:, 4:].isnan().any()
    assert q3.device_status() == 0


def test_values_near_the_end_of_the_range(q3):
    """bf16 values whose weighted sums would pass the range while the maximum lags: the result is finite, in whole and in
    shared items."""
    for n, rows in ((300, 300), (2000, 20)):
        p = Paged([n], 2, 16, BF16, seed=133).fill(134)
        page, slot = p.where(0, range(n))
        p.v[page, :, slot, 11] = 3e36
        ramp = torch.arange(n, device="cuda")[:, None] * (0.02 if n == 300 else 0.003)    # later keys score higher
        p.k[page, :, slot, 0] = ramp.to(BF16)
        q = queries(rows, 8, BF16, 135)
        q[:, :, 0] = 8.0
        got = q3.attention_prompt(*p.handles([0, rows]), q)
        assert torch.isfinite(got).all()
        check_attention(got, q, *p.rows(0), range(n - rows + 1, n + 1), BF16, H)
    assert q3.device_status() == 0


@pytest.mark.parametrize("n,rows", [(300, 300), (2000, 20)])
def test_f32_elements_that_their_parts_do_not_hold(q3, n, rows):
    """Elements that round to infinity in bf16: a value, and queries against keys that are as small."""
    p = Paged([n], 2, 16, F32, seed=136).fill(137)
    page, slot = p.where(0, range(n))
    at = n - rows // 2
    p.v[page[at], 1, slot[at], 11] = 3.4e38
    p.k[page, :, slot, 0] *= 3e-38
    q = queries(rows, 8, F32, 138)
    q[::2, :, 0] = 3.4e38
    got = q3.attention_prompt(*p.handles([0, rows]), q)
    check_attention(got, q, *p.rows(0), range(n - rows + 1, n + 1), F32)
    assert torch.isfinite(got).all() and q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,rows,at", [(300, 300, 200), (2000, 20, 1990)])
def test_seen_and_hidden_nans(q3, dtype, n, rows, at):
    """A NaN that every row sees in one column and one that only the rows from `at` on see in another."""
    p = Paged([n], 2, 16, dtype, seed=139).fill(140)
    page, slot = p.where(0, [0, at])
    p.v[page[0], :, slot[0], 3] = NAN
    p.v[page[1], :, slot[1], 50] = NAN
    q = queries(rows, 8, dtype, 141)
    got = q3.attention_prompt(*p.handles([0, rows]), q).double()
    sees = torch.arange(n - rows, n, device="cuda") >= at
    assert got[:, :, 3].isnan().all() and got[sees][:, :, 50].isnan().all()
    k, v = p.rows(0)
    v[0, :, 3] = v[at, :, 50] = 0.0
    want = attend(q.double(), k, v, range(n - rows + 1, n + 1))[0]
    got[:, :, 3] = want[:, :, 3]
    got[sees, :, 50] = want[sees][:, :, 50]
    check_attention(got, q, k, v, range(n - rows + 1, n + 1), dtype, rounding(dtype))
    assert q3.device_status() == 0


def mean_error(got, want):
    return float((got.double() - want).abs().mean() / want.abs().mean())


def parts(x, count):
    """x (binary64) rounded to a sum of `count` bf16."""
    left, total = x.clone(), torch.zeros_like(x)
    for _ in range(count):
        part = left.to(BF16).double()
        total, left = total + part, left - part
    return total


@pytest.mark.parametrize("n,rows", [(1, 1), (64, 64), (513, 40), (1500, 600), (4096, 40), (4096, 600)])
def test_f32_results_keep_all_their_parts(q3, n, rows):
    """f32 results within 1e-6 = 17 u of the formula on average.  Roundings to nearest average out: a score's chains of at
    most 128 products and the exponential move a weight by some 10 u, the sums of the weighted values, at most n / 64
    tiles one after the other, by sqrt(n / 64) u.  A third bf16 part that is lost from an operand does not pass: it costs
    some 2e-6 = 34 u, as the oracle shows."""
    p = Paged([n], 2, 16, F32, seed=142).fill(143)
    q = queries(rows, 8, F32, 144)
    (k, v), seen = p.rows(0), range(n - rows + 1, n + 1)
    want = attend(q.double(), k, v, seen)[0]
    assert mean_error(q3.attention_prompt(*p.handles([0, rows]), q), want) < 1e-6
    assert mean_error(q3.attention_paged(*p.handles(), q[-1:]), want[-1:]) < 1e-6
    assert mean_error(attend(q.double(), k, parts(v, 2), seen)[0], want) > 1.2e-6
    if n > 1:
        assert mean_error(attend(parts(q.double(), 2), k, v, seen)[0], want) > 1.2e-6
    b = Paged([n], 2, 16, BF16, seed=145).fill(146)
    k, v = b.rows(0)
    one = attend(q[-1:].double(), k, v, [n])[0]
    assert mean_error(q3.attention_paged(*b.handles(), q[-1:]), one) < 1e-6


@pytest.mark.parametrize("cache_t", [F32, BF16])
@pytest.mark.parametrize("heads,n_kv", [(7, 1), (9, 1), (11, 1), (26, 2), (45, 3)])
def test_odd_groups(q3, cache_t, heads, n_kv):
    """Groups of query heads that fill neither a tile's 128 rows nor a product's eight columns."""
    rows, lens = [70, 33, 0, 5, 1], [700, 33, 0, 64, 1]
    p = Paged(lens, n_kv, 32, cache_t, seed=147).fill(148)
    off = offsets(rows)
    for io in (F32, BF16):
        q = queries(5, heads, io, 149)
        got = q3.attention_paged(*p.handles(), q)
        for s, n in enumerate(lens):
            check_attention(got[s:s + 1], q[s:s + 1], *p.rows(s), [n], io)
    q = queries(off[-1], heads, cache_t, 150)
    got = q3.attention_prompt(*p.handles(off), q)
    for s, (r, n) in enumerate(zip(rows, lens)):
        mine = slice(off[s], off[s + 1])
        if r:
            check_attention(got[mine], q[mine], *p.rows(s), range(n - r + 1, n + 1), cache_t, rounding(cache_t))
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_thousands_of_sequences(q3, dtype):
    """Prompts of one to three rows and empty ones, thousands of them: results, and a time that grows with their number and
    not with its square."""
    from metalqwen3_b200.q3cu import KVBatch, KVCache
    k, v = (queries(64 * 16, 2, dtype, s).view(64, 16, 2, 128).transpose(1, 2).contiguous() for s in (151, 152))
    cache, usual = KVCache(k, v), []
    for n in (2500, 20000):
        rows = torch.arange(n) % 4
        off = torch.cat([torch.zeros(1, dtype=torch.long), rows.cumsum(0)])
        lens = rows + torch.arange(n) % 13
        table = (torch.arange(n) * 7 % 64)[:, None]
        batch = KVBatch(*(t.int().cuda() for t in (lens, table, off)))
        q = queries(int(off[-1]), 4, dtype, 153)
        got = q3.attention_prompt(cache, batch, q)
        times = []
        for _ in range(4):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            q3.attention_prompt(cache, batch, q, out=got)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        usual.append(min(times))
        for s in list(range(0, n, n // 37)) + [n - 1]:
            a, b, page, m = int(off[s]), int(off[s + 1]), int(table[s]), int(lens[s])
            if b > a:
                check_attention(got[a:b], q[a:b], k[page].transpose(0, 1)[:m].double(), v[page].transpose(0, 1)[:m].double(),
                                range(m - (b - a) + 1, m + 1), dtype, rounding(dtype))
    assert usual[1] < 24 * usual[0], usual                   # 8 times the sequences
    assert q3.device_status() == 0


def test_empty_slots_between_sequences(q3):
    """Runs of tiles that go from one sequence over thousands of empty ones to the next."""
    from metalqwen3_b200.q3cu import KVBatch, KVCache
    n, pages = 30000, 40
    k, v = (queries(64 * 16, 2, BF16, s).view(64, 16, 2, 128).transpose(1, 2).contiguous() for s in (155, 156))
    table = (torch.arange(n)[:, None] * 5 + torch.arange(pages)) % 64
    q = queries(n, 4, BF16, 157)
    for busy in ([0, 1, 31, 32, 33, 20000, 29999], list(range(300)) + list(range(29700, 30000))):
        lens = torch.zeros(n, dtype=torch.int32)
        lens[busy] = torch.tensor([640 - 3 * (i % 200) for i in range(len(busy))], dtype=torch.int32)
        got = q3.attention_paged(KVCache(k, v), KVBatch(lens.cuda(), table.int().cuda()), q)
        for s in busy[::max(1, len(busy) // 40)] + [busy[-1]]:
            m = int(lens[s])
            kk, vv = (t[table[s]].transpose(0, 1).reshape(2, -1, 128).transpose(0, 1)[:m].double() for t in (k, v))
            check_attention(got[s:s + 1], q[s:s + 1], kk, vv, [m], BF16)
        assert (got[(lens == 0).cuda()] == 0).all() and not got[(lens > 0).cuda()].isnan().any()
    assert q3.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_items_of_many_sequences(q3, dtype):
    """More sequences than are sorted, few enough items that two multiprocessors share one, slots without rows among them."""
    rows = [i % 3 for i in range(70)]
    lens = [r + 1100 + 13 * i for i, r in enumerate(rows)]
    p = Paged(lens, 1, 64, dtype, seed=158).fill(159)
    off = offsets(rows)
    q = queries(off[-1], 4, dtype, 160)
    got = q3.attention_prompt(*p.handles(off), q)
    for s, (r, n) in enumerate(zip(rows, lens)):
        if r:
            mine = slice(off[s], off[s + 1])
            check_attention(got[mine], q[mine], *p.rows(s), range(n - r + 1, n + 1), dtype, rounding(dtype))
    assert q3.device_status() == 0
