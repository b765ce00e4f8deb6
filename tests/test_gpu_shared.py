"""Attention of one new token per sequence where groups of sequences share their first positions, against the formula in
binary64.  Tolerances as in test_gpu_paged.py for bf16 prompts (a probability is rounded to bf16, 2^-8 relative, at shared
positions; elsewhere to less) and, over a Q8_0 cache, as in test_gpu_paged_q8.py, with the shared positions' elements
rounded as prompts round them.  The join of the parts is one product and one sum in binary32 for each: up to 450
of them, which the (n + 64) u of n positions covers, as every part has one at least."""
import math

import pytest
import torch

from test_gpu_kv_forms import I8, Quantised
from test_gpu_paged import BF16, F32, H, Paged, attend, queries
from test_gpu_paged_q8 import check_attention, rounded

pytestmark = pytest.mark.gpu


class Shared:
    """Groups of sequences on one pool: `groups` of (sequences, shared positions), own positions behind them."""

    def __init__(self, groups, own, n_kv, page, q8, seed, complete=True, gap=0):
        self.sizes, self.shared = [g[0] for g in groups], [g[1] for g in groups for _ in range(g[0])]
        self.lens = [a + b for a, b in zip(self.shared, own)]
        self.page, self.q8, self.groups = page, q8, groups
        p = self.p = (Quantised(self.lens, n_kv, page, seed=seed, gap=gap) if q8
                      else Paged(self.lens, n_kv, page, BF16, seed=seed, gap=gap)).fill(seed + 1)
        first = 0
        for size, shared in groups:
            for s in range(first + 1, first + size):
                whole, rest = shared // page, shared % page
                if rest:                        # a page that is shared in part: its first slots again in the own page
                    a, b = int(p.table[first, whole]), int(p.table[s, whole])
                    for t in ([p.k, p.v] + ([p.ks, p.vs] if q8 else [])):
                        t[b, :, :rest] = t[a, :, :rest]
                p.table[s, :whole] = p.table[first, :whole] if complete else -5
            first += size

    def prefix(self, lens=None):
        from metalqwen3_b200.q3cu import KVPrefix
        off = torch.tensor([0] + self.sizes, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        return KVPrefix(off.cuda(), torch.tensor(lens or [g[1] for g in self.groups], dtype=torch.int32, device="cuda"))

    def rows(self, s):
        """Keys and values as the operator takes them."""
        first = sum(self.sizes[:next(i for i in range(len(self.sizes)) if sum(self.sizes[:i + 1]) > s)])
        n = self.shared[s] if self.lens[s] >= self.shared[s] and self.sizes[self.sizes.index(
            next(z for i, z in enumerate(self.sizes) if sum(self.sizes[:i + 1]) > s))] > 1 else 0
        own, lead = self.p.rows(s), rounded(self.p, first) if self.q8 else self.p.rows(first)
        return tuple(torch.cat([a[:n], b[n:]]) for a, b in zip(lead, own))

    def check(self, got, q, which=None):
        for s in which if which is not None else range(len(self.lens)):
            check_attention(got[s:s + 1], q[s:s + 1], *self.rows(s), [self.lens[s]], BF16, H)


def check_average(sh, got, q):
    """The root mean square of all errors.  Rounding the result and the probabilities to bf16 moves each by up to 2^-8 of
    itself, and if evenly spread by 2^-8 / sqrt(3) on average: the two together by 2^-8 sqrt(2 / 3) = 0.0032 of the results'
    average where, as here, probabilities and values are independent; the rest is far below.  A key too many or too few
    among a thousand shows."""
    want = torch.cat([attend(q[s:s + 1].double(), *sh.rows(s), [n])[0] for s, n in enumerate(sh.lens)])
    assert (got.double() - want).pow(2).mean().sqrt() <= 0.0033 * want.pow(2).mean().sqrt() + 1e-30


CASES = [
    # groups of (sequences, shared positions); positions behind them
    (32, 8, 64, [(5, 700)], [1, 90, 64, 33, 7]),
    (16, 8, 16, [(2, 16)], [1, 200]),
    (8, 8, 128, [(3, 128)], [0, 1, 0]),                                       # nothing of their own
    (40, 8, 16, [(1, 300), (4, 129), (2, 1)], [5, 3, 0, 40, 100, 7, 9]),      # one alone; one position shared
    (64, 8, 32, [(40, 1000)], [1 + i * 3 for i in range(40)]),                # several blocks of sequences
    (16, 1, 256, [(7, 2000), (9, 0), (3, 513)], [10 + i for i in range(19)]),  # nothing shared in the second
    (12, 4, 64, [(100, 77)], [i % 5 for i in range(100)]),
    (10, 2, 16, [(3, 260)], [300, 17, 2]),
    (32, 8, 64, [(64, 4096)], [1] * 64),
    (3, 1, 16, [(70, 50), (70, 33), (3, 999)], [2] * 143),
]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("heads,n_kv,page,groups,own", CASES)
def test_attention_shared(q3, q8, heads, n_kv, page, groups, own):
    """Tables whose later sequences have no entries for the pages that are shared whole."""
    sh = Shared(groups, own, n_kv, page, q8, seed=11, complete=False)
    q = queries(len(own), heads, BF16, 13)
    cache, batch = sh.p.handles()
    out = torch.full((len(own), heads, 128), 7.0, dtype=BF16, device="cuda")
    assert q3.attention_shared(cache, batch, sh.prefix(), q, out=out) is out
    assert q3.device_status() == 0
    if any(n == 1 and s for n, s in groups):    # a sequence alone attends to its own pages, which are all there
        assert int(sh.p.table[0, 0]) >= 0
    sh.check(out, q)
    check_average(sh, out, q)


@pytest.mark.parametrize("q8", [False, True])
def test_the_same_as_one_token_attention(q3, q8):
    """Complete tables: attention_paged gives the same but for the rounding; and so does a call without groups."""
    from metalqwen3_b200.q3cu import KVPrefix
    sh = Shared([(6, 333), (5, 100)], [3 * i for i in range(11)], 4, 16, q8, seed=20)
    q = queries(11, 16, BF16, 21)
    cache, batch = sh.p.handles()
    sh.check(q3.attention_shared(cache, batch, sh.prefix(), q), q)
    one = q3.attention_paged(cache, batch, q)
    i32 = dict(dtype=torch.int32, device="cuda")
    none = KVPrefix(torch.zeros(1, **i32), torch.zeros(0, **i32))
    plain = q3.attention_shared(cache, batch, none, q)
    for s in range(11):
        check_attention(plain[s:s + 1], q[s:s + 1], *sh.p.rows(s), [sh.lens[s]], BF16, 2.0 ** -11)
        check_attention(one[s:s + 1], q[s:s + 1], *sh.p.rows(s), [sh.lens[s]], BF16, 2.0 ** -11)


@pytest.mark.parametrize("q8", [False, True])
def test_sequences_outside_groups_and_short_ones(q3, q8):
    """Groups over a part of the batch; a sequence that holds less than is shared, empty ones, and padding."""
    from metalqwen3_b200.q3cu import KVPrefix
    sh = Shared([(8, 200)], [0, 10, 20, 30, 40, 50, 60, 70], 2, 16, q8, seed=22)
    i32 = dict(dtype=torch.int32, device="cuda")
    prefix = KVPrefix(torch.tensor([2, 6], **i32), torch.tensor([150], **i32))
    p = sh.p
    p.lens = [200, 210, 220, 149, 150, 0, 260, 270]
    p.kv_len.copy_(torch.tensor(p.lens[:5] + [-3] + p.lens[6:], dtype=torch.int32))
    q = queries(8, 8, BF16, 23)
    got = q3.attention_shared(*p.handles(), prefix, q)
    assert q3.device_status() == 0 and (got[5] == 0).all()
    for s in (0, 1, 2, 3, 4, 6, 7):
        k, v = p.rows(s)
        if s in (2, 4) and q8:
            k, v = (torch.cat([a[:150], b[150:]]) for a, b in zip(rounded(p, s), (k, v)))
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [p.lens[s]], BF16, H)


def test_bad_groups_and_pages(q3):
    """Offsets that do not rise or leave the batch share nothing; a bad page of the shared part reads as zeros for all of
    the group, a length beyond the table is cut; both are flagged."""
    from metalqwen3_b200.q3cu import DEV_BAD_INDEX, KVPrefix
    i32 = dict(dtype=torch.int32, device="cuda")
    sh = Shared([(6, 100)], [9, 8, 7, 6, 5, 4], 2, 16, False, seed=24)
    q = queries(6, 4, BF16, 25)
    cache, batch = sh.p.handles()
    for off in ([0, 7], [-1, 3], [4, 4], [5, 2]):
        got = q3.attention_shared(cache, batch, KVPrefix(torch.tensor(off, **i32), torch.tensor([100], **i32)), q)
        assert q3.device_status() == 0
        for s in range(6):
            check_attention(got[s:s + 1], q[s:s + 1], *sh.p.rows(s), [sh.lens[s]], BF16, H)
    sh.p.table[0, 2] = 1 << 30
    got = q3.attention_shared(cache, batch, sh.prefix(), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    for s in range(6):
        k, v = sh.p.rows(s) if s else sh.p.rows(1)
        if s == 0:
            own = slice(100, sh.lens[0])
            page, slot = sh.p.where(0, range(100, sh.lens[0]))
            k, v = (torch.cat([a[:100], t[page, :, slot].double()]) for a, t in ((k, sh.p.k), (v, sh.p.v)))
        k, v = k.clone(), v.clone()
        k[32:48] = v[32:48] = 0
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [sh.lens[s]], BF16, H)
    cap = sh.p.max_pages * 16
    sh.p.table[:] = sh.p.table[1, 0]
    sh.p.kv_len[:] = cap + 5
    got = q3.attention_shared(cache, batch, sh.prefix([cap + 1]), q)
    assert q3.device_status() == DEV_BAD_INDEX and q3.device_status() == 0
    again = torch.arange(cap, device="cuda") % 16
    page = sh.p.table[1, 0].long()
    k, v = (t[page].double().transpose(0, 1)[again] for t in (sh.p.k, sh.p.v))
    for s in range(6):
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [cap], BF16, H)


@pytest.mark.parametrize("q8", [False, True])
def test_strides_work_and_streams(q3, q8):
    """Pages further apart than they are large, queries inside wider rows, a workspace of any contents and for more
    sequences, two calls at once on two streams."""
    sh = Shared([(9, 500)], list(range(9)), 4, 32, q8, seed=26, gap=4096 + 32)
    wide = queries(9, 48, BF16, 27)
    q = wide[:, 8:24]
    cache, batch = sh.p.handles()
    prefix = sh.prefix()
    works = [torch.full((q3.attention_shared_workspace(cache, n, 16).numel(),), 255, dtype=torch.uint8, device="cuda") for n in (9, 30)]
    outs = [torch.empty((9, 16, 128), dtype=BF16, device="cuda") for _ in works]
    streams = [torch.cuda.Stream() for _ in works]
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, work, out in zip(streams, works, outs):
            with torch.cuda.stream(stream):
                assert q3.attention_shared(cache, batch, prefix, q, out=out, work=work) is out
    torch.cuda.synchronize()
    for out in outs:
        sh.check(out, q)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], q3.attention_shared(cache, batch, prefix, q))
    assert q3.device_status() == 0


@pytest.mark.parametrize("q8", [False, True])
def test_a_serving_step_as_a_graph(q3, q8):
    """Append, then attention behind the shared prefix, captured and replayed while sequences grow and groups change."""
    from metalqwen3_b200.q3cu import KVPrefix, Rope
    own = [20, 3, 40, 1, 9]
    sh = Shared([(5, 96)], [x + 40 for x in own], 2, 16, q8, seed=28)
    p, heads, n_kv = sh.p, 8, 2
    qkv = queries(5, heads + 2 * n_kv, F32, 29)
    cache, batch = p.handles(list(range(6)))
    i32 = dict(dtype=torch.int32, device="cuda")
    off, length = torch.tensor([0, 5, 5], **i32), torch.tensor([96, 0], **i32)
    prefix = KVPrefix(off, length)
    work = q3.attention_shared_workspace(cache, 5, heads)
    q_out, out = (torch.empty((5, heads, 128), dtype=BF16, device="cuda") for _ in range(2))
    rope = Rope(theta=1e4, interleaved=True)

    def step():
        q3.kv_append(cache, batch, qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:], q_out=q_out, rope=rope)
        q3.attention_shared(cache, batch, prefix, q_out, out=out, work=work)
    p.kv_len.copy_(torch.tensor([96 + x for x in own], dtype=torch.int32))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for n, offs, lens in ((1, [0, 5, 5], [96, 0]), (2, [0, 2, 5], [96, 64]), (40, [1, 3, 5], [32, 96])):
        now = [96 + x + n for x in own]
        p.kv_len.copy_(torch.tensor(now, dtype=torch.int32))
        off.copy_(torch.tensor(offs, dtype=torch.int32))
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        qkv.copy_(queries(5, heads + 2 * n_kv, F32, 30 + n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        p.lens = now
        for s in range(5):
            g = next((i for i in range(2) if offs[i] <= s < offs[i + 1]), None)
            k, v = p.rows(s)
            if q8 and g is not None:
                k, v = (torch.cat([a[:lens[g]], b[lens[g]:]]) for a, b in zip(rounded(p, s), (k, v)))
            check_attention(out[s:s + 1], q_out[s:s + 1], k, v, [now[s]], BF16, H)
    assert q3.device_status() == 0


def test_far_positions_pass_32_bits(q3):
    """A shared part of 200,000 positions on few pages, page starts beyond 2^31 elements."""
    from metalqwen3_b200.q3cu import KVBatch, KVCache, KVPrefix
    gap, page, n = (1 << 29), 256, 200_000
    pool = [torch.zeros(8 * gap + page * 128, dtype=BF16, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((9, 1, page, 128), (gap, page * 128, 128, 1)) for t in pool)
    for i in range(9):
        k[i], v[i] = queries(page, 1, BF16, i).view(1, page, 128), queries(page, 1, BF16, 20 + i).view(1, page, 128)
    pages = -(-(n + 50) // page)
    table = (torch.arange(pages) % 9).int().repeat(3, 1).cuda()
    lens = [n, n + 1, n + 50]
    i32 = dict(dtype=torch.int32, device="cuda")
    q = queries(3, 4, BF16, 50)
    got = q3.attention_shared(KVCache(k, v), KVBatch(torch.tensor(lens, **i32), table), KVPrefix(torch.tensor([0, 3], **i32),
                              torch.tensor([n], **i32)), q)
    assert q3.device_status() == 0
    at = torch.arange(n + 50, device="cuda")
    kk, vv = (t[table[0, at // page].long(), :, at % page].double() for t in (k, v))
    for s in range(3):
        check_attention(got[s:s + 1], q[s:s + 1], kk[:lens[s]], vv[:lens[s]], [lens[s]], BF16, H)


@pytest.mark.parametrize("q8", [False, True])
def test_more_groups_than_threads(q3, q8):
    """1,300 groups (the plan's CTA has 1,024 threads) of 2,700 sequences, many of which share nothing or hold nothing."""
    from metalqwen3_b200.q3cu import KVPrefix
    n = 2700
    p = (Quantised([20] * n, 1, 16, seed=40) if q8 else Paged([20] * n, 1, 16, BF16, seed=40)).fill(41)
    gen = torch.Generator().manual_seed(42)
    lens = torch.randint(0, 21, (n,), generator=gen).int()
    first = torch.arange(1301).int() * 2 + 50                 # pairs, from sequence 50 on
    shared = torch.randint(0, 21, (1300,), generator=gen).int()
    lead, other = first[:-1].long(), first[:-1].long() + 1
    for t in [p.k, p.v] + ([p.ks, p.vs] if q8 else []):       # the second holds the same positions on its own pages
        for i in range(2):
            t[p.table[other.cuda(), i].long()] = t[p.table[lead.cuda(), i].long()]
    p.kv_len.copy_(lens)
    q = queries(n, 2, BF16, 43)
    cache, batch = p.handles()
    got = q3.attention_shared(cache, batch, KVPrefix(first.cuda(), shared.cuda()), q).double()
    assert q3.device_status() == 0
    want = q3.attention_paged(cache, batch, q).double()
    empty = (lens == 0).cuda()
    assert empty.any() and (got[empty] == 0).all() and torch.isfinite(got).all()
    p.lens = lens.tolist()
    group = {int(x): i // 2 for i, x in enumerate(torch.stack([lead, other], 1).flatten())}
    active = [s for s in range(n) if s in group and 0 < shared[group[s]] <= min(lens[s], lens[lead[group[s]]])]
    assert len(active) > 500
    for s in active[::7]:
        m, k, v = int(shared[group[s]]), *p.rows(s)
        if q8:
            k, v = (torch.cat([a[:m], b[m:]]) for a, b in zip(rounded(p, int(lead[group[s]])), (k, v)))
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [p.lens[s]], BF16, H)
    # In no group, or in one that shares nothing: attention_paged's result, cut into other runs, so that a weight is rounded
    # elsewhere (2^-11 in each) and the result with it (2^-8 in each).
    alone = torch.tensor([s not in group or not shared[group[s]] for s in range(n)]).cuda()
    top = max(float(p.rows(s)[1].abs().max()) for s in range(n) if p.lens[s])
    assert ((got - want)[alone].abs() <= 1.01 * (2 * 2.0 ** -8 * want[alone].abs() + 4 * 2.0 ** -11 * top)).all()


@pytest.mark.parametrize("q8", [False, True])
def test_calls_one_after_the_other(q3, q8):
    """Calls on one workspace and one result, queries, lengths and groups changed between them by kernels of the same
    stream, nothing waited for: each gives what it gives by itself."""
    from metalqwen3_b200.q3cu import KVPrefix
    sh = Shared([(6, 700), (5, 300)], [20 * i for i in range(11)], 4, 16, q8, seed=44)
    p = sh.p
    cache, batch = p.handles()
    i32 = dict(dtype=torch.int32, device="cuda")
    off, length = torch.tensor([0, 6, 11], **i32), torch.tensor([700, 300], **i32)
    prefix = KVPrefix(off, length)
    work = q3.attention_shared_workspace(cache, 11, 16)
    out, q = (torch.empty((11, 16, 128), dtype=BF16, device="cuda") for _ in range(2))
    ways = []
    for i, (offs, lens, cut) in enumerate([([0, 6, 11], [700, 300], 0), ([0, 3, 6], [512, 700], 15), ([2, 6, 11], [1, 256], 40),
                                           ([0, 0, 0], [5, 5], 3)]):
        ways.append((torch.tensor(offs, **i32), torch.tensor(lens, **i32), p.kv_len - cut, queries(11, 16, BF16, 45 + i)))

    def call(way):
        for to, x in zip((off, length, p.kv_len, q), way):
            to.copy_(x)
        q3.attention_shared(cache, batch, prefix, q, out=out, work=work)
        return out.clone()
    alone = []
    for way in ways:
        torch.cuda.synchronize()
        alone.append(call(way))
    torch.cuda.synchronize()
    got = [(i, call(ways[i])) for _ in range(30) for i in (0, 1, 2, 3, 1, 0, 2)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone[i]) for i, x in got)
    assert q3.device_status() == 0


def test_wild_groups(q3):
    """Thousands of groups whose offsets jump about: what they share is anyone's guess, but nothing faults, and the next
    call is right."""
    from metalqwen3_b200.q3cu import KVPrefix
    sh = Shared([(40, 60), (60, 33)], [3] * 100, 2, 16, False, seed=46)
    cache, batch = sh.p.handles()
    q = queries(100, 4, BF16, 47)
    gen = torch.Generator().manual_seed(48)
    for high in (101, 3, 1 << 30):
        off = torch.randint(-2, high, (3001,), generator=gen).int().cuda()
        length = torch.randint(-5, 64, (3000,), generator=gen).int().cuda()
        q3.attention_shared(cache, batch, KVPrefix(off, length), q)
    assert q3.device_status() == 0
    sh.check(q3.attention_shared(cache, batch, sh.prefix(), q), q)


def test_nan_and_peaked(q3):
    """Scores in the thousands and all equal; a NaN value in the shared part shows in its column of every row, one of a
    sequence's own only there; what lies behind a length (NaN) reaches nothing."""
    for scale in (60.0, 0.0):
        sh = Shared([(4, 400)], [30, 1, 0, 77], 2, 16, False, seed=31)
        q = queries(4, 8, BF16, 32, scale)
        sh.check(q3.attention_shared(*sh.p.handles(), sh.prefix(), q), q)
    clean = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    page, slot = sh.p.where(3, [450])
    sh.p.v[page, 1, slot, 5] = math.nan
    got = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    assert torch.isnan(got[3, 4:, 5]).all() and torch.equal(got[:3], clean[:3]) and torch.isfinite(got[3, :4]).all()
    page, slot = sh.p.where(0, [399])
    sh.p.v[page, 0, slot, 7] = math.nan
    got = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    assert torch.isnan(got[:, :4, 7]).all() and torch.equal(got[:3, 4:], clean[:3, 4:])


def test_refusals(q3):
    from metalqwen3_b200.q3cu import KVPrefix, Q3Error
    sh = Shared([(3, 40)], [1, 2, 3], 2, 16, False, seed=33)
    cache, batch = sh.p.handles()
    prefix, q = sh.prefix(), queries(3, 4, BF16, 34)

    def refused(status, call):
        with pytest.raises(Q3Error) as e:
            call()
        assert e.value.status == status

    wide = Paged([20, 20, 20], 2, 16, F32, seed=35)
    refused(1, lambda: q3.attention_shared(cache, batch, prefix, q.float()))
    refused(1, lambda: q3.attention_shared(*wide.handles(), prefix, q))
    refused(1, lambda: q3.attention_shared(cache, batch, prefix, q, out=q))
    refused(1, lambda: q3.attention_shared(cache, batch, prefix, q, work=torch.empty(64, dtype=torch.uint8, device="cuda")))
    refused(1, lambda: q3.attention_shared(cache, batch, prefix, queries(3, 3, BF16, 34)))
    refused(1, lambda: q3.attention_prompt(*Quantised([20], 2, 16, seed=36).handles([0, 1]), queries(1, 4, F32, 37)))
    with pytest.raises(ValueError):
        KVPrefix(prefix.seq_off, prefix.length.repeat(2))
    with pytest.raises(TypeError):
        KVPrefix(prefix.seq_off.long(), prefix.length)
    assert q3.device_status() == 0
