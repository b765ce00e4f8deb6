"""Which sequences of a group share what, where lengths and offsets are not as they mostly are.  Tolerances as in
test_gpu_shared.py."""
import pytest
import torch

from test_gpu_paged import BF16, H, queries
from test_gpu_paged_q8 import check_attention
from test_gpu_shared import Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("held", [0, 150, -4])
def test_a_first_sequence_that_holds_less_than_is_shared(q3, q8, held):
    """Its slot was freed, say, and its page ids are another sequence's by now: the group shares nothing then, and each
    sequence attends to its own pages.  A group beside it shares as before."""
    sh = Shared([(4, 200), (3, 90)], [10, 20, 30, 40, 5, 6, 7], 2, 16, q8, seed=51)
    p = sh.p
    p.table[0, :13] = p.table[3, :13].flip(0)           # stale, and of other positions
    p.kv_len[0] = held
    q = queries(7, 8, BF16, 52)
    got = q3.attention_shared(*p.handles(), sh.prefix(), q)
    assert q3.device_status() == 0
    for s in (1, 2, 3):
        check_attention(got[s:s + 1], q[s:s + 1], *p.rows(s), [sh.lens[s]], BF16, H)
    sh.check(got, q, (4, 5, 6))
    if held > 0:
        p.lens[0] = held
        check_attention(got[:1], q[:1], *p.rows(0), [held], BF16, H)
    else:
        assert (got[0] == 0).all()


def test_groups_that_overlap(q3):
    """Offsets that fall make two groups claim the same sequences: each sequence attends behind one first sequence, the one
    whose group the plan finds it in, and no other group writes its results.  The long third group makes runs of several
    items, so that the second group's results are written behind the first's."""
    from metalqwen3_b200.q3cu import KVPrefix
    i32 = dict(dtype=torch.int32, device="cuda")
    sh = Shared([(4, 96), (2, 96), (2, 50_000)], [10 + i for i in range(8)], 2, 16, False, seed=53)
    p = sh.p
    q = queries(8, 32, BF16, 54)
    # sequences 0 .. 3, again 2 .. 5 (of which 2 and 3 are the first group's), and 6, 7
    prefix = KVPrefix(torch.tensor([0, 0, 4, 2, 6, 8], **i32), torch.tensor([0, 96, 0, 96, 50_000], **i32))
    p.table[2, :6] = p.table[4, :6].flip(0)           # what sequence 2 has there is its own
    got = q3.attention_shared(*p.handles(), prefix, q)
    assert q3.device_status() == 0
    for s in range(8):
        first = 0 if s < 4 else 2 if s < 6 else 6
        n = 96 if s < 6 else 50_000
        own, lead = p.rows(s), p.rows(first)
        k, v = (torch.cat([a[:n], b[n:]]) for a, b in zip(lead, own))
        check_attention(got[s:s + 1], q[s:s + 1], k, v, [sh.lens[s]], BF16, H)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("page,shared", [(16, 200), (64, 200), (256, 500)])
def test_first_slots_of_a_page_that_is_shared_in_part(q3, q8, page, shared):
    """The shared positions on a sequence's own page are the first sequence's to hold: NaN there (in a Q8_0 cache's scales)
    reaches nothing."""
    sh = Shared([(5, shared)], [1, 60, 3, 300, 2], 2, page, q8, seed=55)
    q = queries(5, 8, BF16, 56)
    clean = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    for s in range(1, 5):
        b = int(sh.p.table[s, shared // page])
        for t in (sh.p.ks, sh.p.vs) if q8 else (sh.p.k, sh.p.v):
            t[b, :, :shared % page] = float("nan")
    assert torch.equal(q3.attention_shared(*sh.p.handles(), sh.prefix(), q), clean)
    for s in range(1, 5):                                # (the formula takes the first sequence's)
        a, b = int(sh.p.table[0, shared // page]), int(sh.p.table[s, shared // page])
        for t in (sh.p.ks, sh.p.vs) if q8 else (sh.p.k, sh.p.v):
            t[b, :, :shared % page] = t[a, :, :shared % page]
    sh.check(clean, q)
    assert q3.device_status() == 0
