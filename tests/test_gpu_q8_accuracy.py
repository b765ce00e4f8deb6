"""Prompts and shared positions over a Q8_0 cache against what the cache holds: products of codes and scales that are not
rounded, in binary64.  (test_gpu_paged_q8.py takes them as the kernels round them.)

Largest errors.  A key or value element is rounded twice to 11 bits, its scale and the product: by 2 W + W^2 of itself, W = 2^-11.
So a score is off by that share of A = sum |q_i k_i| / sqrt(128), beside the terms of test_gpu_paged_q8.py, a softmax weight by a
factor e^(2 ds), and a value's part of the result by 2 W + W^2 again; a probability by W, or 2^-32.

Average errors.  Roundings to 11 bits move a number by no more than W of itself, evenly spread: a mean square of at most
E = W^2 / 3 of its square (half of that over numbers evenly spread in their logarithm, which leaves more than chance needs).  The error of
a scale is common to its 64 elements, all others are independent.  With S_0 and S_1 the two halves' parts of a score, its variance is
at most E (S_0^2 + S_1^2 + sum (q_i k_i)^2 / 128), and that of a result
    sum_t p_t^2 (3 E v_t^2 + var(s_t) (v_t - o)^2)
for one rounding of the probability and two of the value.  The rounding of the result itself is known: that of o to bf16.  Were
probabilities rounded to bf16, the errors would be above all that where many positions have their share of the weight, which the tests
show with the formula.
"""
import math

import pytest
import torch

from test_gpu_paged import BF16, H, U, attend, offsets, queries
from test_gpu_kv_forms import Quantised
from test_gpu_paged_q8 import W, check_attention as check_exact
from test_gpu_shared import Shared

pytestmark = pytest.mark.gpu
W2, E = 2 * W + W * W, W * W / 3
FREE = [i for i in range(128) if i != 5]      # dimensions of independent values: all codes of dimension 5 are -128


def check_largest(got, q, k, v, seen):
    o, pv, a = attend(q.double(), k, v, seen)
    n = k.shape[0]
    ds = (160 * U + W2) * a + math.sqrt(128) * 2.0 ** -39 * float(q.abs().max()) * float(k.abs().max())
    tol = (torch.expm1(2 * ds) + (n + 64) * U + W + W2) * pv + n * (2.0 ** -32 + 2.0 ** -39) * 1.01 * float(v.abs().max())
    tol = tol + H * (o.abs() + tol)
    assert ((got.double() - o).abs() <= tol).all()


def average(got, q, k, v, seen, sums=(0.0, 0.0, 0.0)):
    """Sums of squares: of the errors, of what they may be, and of what they were with probabilities in bf16 alone."""
    square, bound, planted = sums
    for i, m in enumerate(seen):
        for h in range(q.shape[1]):
            kk, vv = (t[:m, h * t.shape[1] // q.shape[1]] for t in (k, v))
            x = q[i, h].double()
            part = kk * x / math.sqrt(128)
            score = part.sum(-1)
            p = torch.softmax(score, 0)
            o = p @ vv
            var_s = E * (part[:, :64].sum(-1) ** 2 + part[:, 64:].sum(-1) ** 2 + (part ** 2).sum(-1))
            var = (p * p) @ (3 * E * vv ** 2 + var_s[:, None] * (vv - o) ** 2)
            square = square + ((got[i, h].double() - o) ** 2)[FREE].sum()
            bound = bound + (var + (o.bfloat16().double() - o) ** 2)[FREE].sum()
            w = torch.exp(score - score.max())
            planted = planted + (((w.bfloat16().double() @ vv / w.sum()).bfloat16().double() - o) ** 2)[FREE].sum()
    return square, bound, planted


@pytest.mark.parametrize("scale", [1.5, 0.5])
@pytest.mark.parametrize("heads,n_kv,page,rows,lens", [(32, 8, 64, [300, 40], [300, 900]), (3, 1, 16, [20], [5000]),
                                                       (16, 1, 32, [130], [130]), (8, 8, 128, [5, 77, 0], [2000, 500, 10])])
def test_prompts(q3, scale, heads, n_kv, page, rows, lens):
    p = Quantised(lens, n_kv, page, seed=90).fill(91)
    q = queries(sum(rows), heads, BF16, 92, scale)
    got = q3.attention_prompt(*p.handles(offsets(rows)), q)
    first, sums = 0, (0.0, 0.0, 0.0)
    for s, (r, n) in enumerate(zip(rows, lens)):
        if r:
            mine, seen = slice(first, first + r), range(n - r + 1, n + 1)
            check_largest(got[mine], q[mine], *p.rows(s), seen)
            some = range(0, r, 1 + r // 20)
            sums = average(got[mine][some], q[mine][some], *p.rows(s), [seen[i] for i in some], sums)
        first += r
    assert sums[0] <= sums[1] and (scale > 1 or sums[1] < sums[2]) and q3.device_status() == 0


@pytest.mark.parametrize("scale", [1.5, 0.5])
@pytest.mark.parametrize("heads,n_kv,page,groups,own", [(32, 8, 64, [(5, 700)], [1, 90, 64, 33, 7]),
                                                       (16, 2, 16, [(12, 1500), (9, 300)], [1 + 2 * i for i in range(21)]),
                                                       (10, 2, 32, [(40, 129)], [1] * 40)])
def test_shared_positions(q3, scale, heads, n_kv, page, groups, own):
    sh = Shared(groups, own, n_kv, page, True, seed=93)
    # (94 is the keys' seed as well: some of the keys are the queries, and weigh most.  At the smaller scale none are.)
    q = queries(len(own), heads, BF16, 94 if scale > 1 else 96, scale)
    got = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    sums = (0.0, 0.0, 0.0)
    for s, n in enumerate(sh.lens):
        check_largest(got[s:s + 1], q[s:s + 1], *sh.p.rows(s), [n])
        sums = average(got[s:s + 1], q[s:s + 1], *sh.p.rows(s), [n], sums)
    assert sums[0] <= sums[1] and (scale > 1 or sums[1] < sums[2]) and q3.device_status() == 0


def test_alone_in_a_group(q3):
    """One sequence shares nothing: its codes are taken exactly, where a group's are rounded, and its weights rounded by W."""
    sh = Shared([(1, 300), (4, 129), (1, 700)], [5, 3, 1, 40, 100, 7], 2, 16, True, seed=97)
    q = queries(6, 16, BF16, 99)
    got = q3.attention_shared(*sh.p.handles(), sh.prefix(), q)
    for s in (0, 5):
        check_exact(got[s:s + 1], q[s:s + 1], *sh.p.rows(s), [sh.lens[s]], BF16, W)
    sh.check(got, q)
    assert q3.device_status() == 0
