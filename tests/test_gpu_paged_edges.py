"""The paged-cache operators where one element, one order or one stream decides.  Formulas, tolerances and helpers are
those of test_gpu_paged.py."""
import pytest
import torch

from test_gpu_paged import BF16, F32, Paged, check_attention, queries

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
