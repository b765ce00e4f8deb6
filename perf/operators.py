"""The paged-cache operators: what is measured, their plain forms and their definitions in 64 bits.

Three operators that a serving step runs one after the other on one layer's paged key-value cache
(pages of [n_kv][page_size][128], one table row of page ids per sequence, packed token rows):

  append   QK-norm and rotation of the packed query and key rows; keys and values into the cache
  prompt   causal attention of packed prompt rows (or of a chunk behind a cached prefix) over the cache
  decode   attention of one new token per sequence over the cache

A case holds sizes only; `layout` derives the ragged lengths from them.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
THETA = 1e6
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_handle = None


def listed():
    return [
        # one sequence's next token behind a full 4096-token prompt: the smallest call, all latency
        dict(name="append_token", op="append", seqs=1, rows=1, prefix=4095, heads=32, kv_heads=8, page=64,
             io="f32", cache="bf16", mix=1),
        # a packed prefill batch of 4096 tokens: the projections' f32 rows in, bf16 queries and cache out
        dict(name="append_prefill", op="append", seqs=6, rows=4096, prefix=0, heads=32, kv_heads=8, page=64,
             io="f32", cache="bf16", mix=2),
        # ragged chunks of prompts behind cached prefixes, everything in f32
        dict(name="append_chunk_f32", op="append", seqs=5, rows=2001, prefix=8192, heads=16, kv_heads=8, page=16,
             io="f32", cache="f32", mix=3),
        # one sequence at position 511 with an f32 cache: single-user decoding
        dict(name="decode_one_f32", op="decode", seqs=1, longest=512, heads=16, kv_heads=8, page=16,
             io="f32", cache="f32", mix=4),
        # a small ragged batch, one slot of it empty
        dict(name="decode_ragged", op="decode", seqs=9, longest=4096, heads=32, kv_heads=8, page=16,
             io="bf16", cache="bf16", mix=5),
        # a full serving batch, lengths spread over 0..16384
        dict(name="decode_batch", op="decode", seqs=64, longest=16384, heads=32, kv_heads=8, page=64,
             io="f32", cache="bf16", mix=6),
        # a single very long context: all the parallelism lies along the cache
        dict(name="decode_long", op="decode", seqs=1, longest=100003, heads=32, kv_heads=8, page=128,
             io="bf16", cache="bf16", mix=7),
        # a short question: latency of the prompt path
        dict(name="prompt_short", op="prompt", seqs=1, rows=37, prefix=0, heads=16, kv_heads=8, page=16,
             io="bf16", cache="bf16", mix=8),
        # a packed prefill batch of 4096 tokens in six prompts
        dict(name="prompt_packed", op="prompt", seqs=6, rows=4096, prefix=0, heads=32, kv_heads=8, page=64,
             io="bf16", cache="bf16", mix=9),
        # ragged chunks behind long cached prefixes (chunked prefill)
        dict(name="prompt_chunk", op="prompt", seqs=4, rows=2043, prefix=8192, heads=32, kv_heads=8, page=64,
             io="bf16", cache="bf16", mix=10),
        # one long document
        dict(name="prompt_long", op="prompt", seqs=1, rows=16384, prefix=0, heads=40, kv_heads=8, page=128,
             io="bf16", cache="bf16", mix=11),
        # an f32 prompt batch
        dict(name="prompt_f32", op="prompt", seqs=3, rows=2000, prefix=0, heads=16, kv_heads=8, page=16,
             io="f32", cache="f32", mix=12),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (40, 8), (8, 8), (64, 8), (12, 4), (16, 1)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]),
                io=rng.choice(["f32", "bf16"]), cache=rng.choice(["f32", "bf16"]), mix=rng.randrange(1, 1 << 20))
    if op == "decode":
        case["seqs"] = _spread(rng, 1, 128)
        case["longest"] = _spread(rng, 1, min(65536, (1 << 19) // case["seqs"]))
        return case
    case["rows"] = _spread(rng, 1, 4096)
    case["seqs"] = _spread(rng, 1, min(64, case["rows"]))
    case["prefix"] = rng.choice([0, 0, _spread(rng, 1, 8192)])
    if op == "prompt":
        case["io"] = case["cache"] = rng.choice(["bf16", "bf16", "f32"])
        if case["io"] == "f32":
            case["rows"] = min(case["rows"], 1024)
            case["seqs"] = min(case["seqs"], case["rows"])
            case["prefix"] = min(case["prefix"], 2048)
    return case


def layout(case):
    """(query rows, cache length with them) of each sequence."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    if case["op"] == "decode":
        lens = [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(n - 1)]
        if n > 4:
            lens[n // 2] = 0                      # an empty slot of the batch
        return [1] * n, lens
    cuts = sorted(rng.sample(range(1, case["rows"]), n - 1)) if n > 1 else []
    rows = [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]
    prefix = [case["prefix"]] + [rng.randint(0, case["prefix"]) for _ in range(n - 1)]
    return rows, [p + r for p, r in zip(prefix, rows)]


def _pairs(case):
    """Scores the mask leaves, per head."""
    return sum(q * kv - q * (q - 1) // 2 for q, kv in zip(*layout(case)))


def work(case):
    rows, lens = layout(case)
    size = {"f32": 4, "bf16": 2}
    io, cache = size[case["io"]], size[case["cache"]]
    total, heads, kv = sum(rows), case["heads"], case["kv_heads"]
    if case["op"] == "append":
        read = total * (heads + 2 * kv) * HEAD_DIM * io
        written = total * (heads + 2 * kv) * HEAD_DIM * cache
        # per query or key element: square and sum, scale and weight, half a rotation
        return {"bytes": read + written, "flops": total * (heads + kv) * HEAD_DIM * 7}
    moved = 2 * total * heads * HEAD_DIM * io + 2 * sum(lens) * kv * HEAD_DIM * cache
    pairs = sum(lens) if case["op"] == "decode" else _pairs(case)
    return {"bytes": moved, "flops": 4 * HEAD_DIM * heads * pairs}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, lens = layout(case)
    n, page, heads, kv = len(rows), case["page"], case["heads"], case["kv_heads"]
    total, io, cache_type = sum(rows), TYPES[case["io"]], TYPES[case["cache"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    max_pages = max(1, max((length + page - 1) // page for length in lens))
    order = random.Random(seed)
    table = torch.full((n, max_pages), -1, dtype=torch.int32)
    # an append touches the pages of its own rows only: its earlier pages are all page 0
    first = [(length - r) // page if case["op"] == "append" else 0 for r, length in zip(rows, lens)]
    used = [(length + page - 1) // page - f for f, length in zip(first, lens)]
    n_pages = 1 + sum(used)
    ids = list(range(1, n_pages))
    order.shuffle(ids)
    for s in range(n):
        table[s, :first[s]] = 0
        table[s, first[s]:first[s] + used[s]] = torch.tensor(ids[:used[s]], dtype=torch.int32)
        del ids[:used[s]]

    def pool():
        out = torch.empty((n_pages, kv, page, HEAD_DIM), dtype=cache_type, device=dev)
        for a in range(0, n_pages, 4096):
            out[a:a + 4096] = normal(min(4096, n_pages - a), kv, page, HEAD_DIM)
        return out

    st = dict(op=case["op"], rows=rows, lens=lens, heads=heads, kv_heads=kv, page=page, k_pages=pool(),
              v_pages=pool(), table=table.to(dev), kv_len=torch.tensor(lens, dtype=torch.int32, device=dev),
              row_off=torch.tensor([0] + rows, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev))
    if case["op"] == "append":
        # the rows of the fused Q|K|V projection, a few channels of it large
        qkv = normal(total, heads + 2 * kv, HEAD_DIM)
        qkv[:, :, 5::50] *= 6.0
        qkv = qkv.to(io)
        st.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv], v=qkv[:, heads + kv:], cache_type=cache_type,
                  q_norm=1 + 0.2 * normal(HEAD_DIM), k_norm=1 + 0.2 * normal(HEAD_DIM),
                  out=torch.empty((total, heads, HEAD_DIM), dtype=cache_type, device=dev))
    else:
        # normalised queries with a little gain, so that the softmax is neither flat nor a single key
        q = normal(total, heads, HEAD_DIM)
        q = 1.5 * q * torch.rsqrt((q * q).mean(-1, keepdim=True))
        st.update(q=q.to(io), out=torch.empty((total, heads, HEAD_DIM), dtype=io, device=dev))
    if own:
        global _handle
        from metalqwen3_b200.q3cu import KVBatch, KVCache, Q3CU
        if _handle is None:
            _handle = Q3CU(0)
        st["q3"] = _handle
        st["cache"] = KVCache(st["k_pages"], st["v_pages"])
        st["batch"] = KVBatch(st["kv_len"], st["table"], st["row_off"])
        if case["op"] == "decode":
            st["space"] = _handle.attention_paged_workspace(st["cache"], heads)
    return st


def run(st):
    if own:
        if st["op"] == "append":
            q = st["q3"].kv_append(st["cache"], st["batch"], st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"],
                                   theta=THETA, eps=EPS, q_out=st["out"])
            return [q, st["k_pages"], st["v_pages"]]
        if st["op"] == "decode":
            return st["q3"].attention_paged(st["cache"], st["batch"], st["q"], out=st["out"], work=st["space"])
        return st["q3"].attention_prompt(st["cache"], st["batch"], st["q"], out=st["out"])
    return _plain_append(st) if st["op"] == "append" else _plain_attention(st)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ------------------

def _plain_rotate(x, weight, pos):
    x = x.float()
    x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * weight
    half = HEAD_DIM // 2
    freq = THETA ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = pos.double()[:, None, None] * freq       # 64 bits: positions reach far past a turn's precision in 32
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_append(st):
    dev = st["q"].device
    seq = torch.cat([torch.full((r,), s, dtype=torch.long, device=dev) for s, r in enumerate(st["rows"])])
    pos = torch.cat([torch.arange(n - r, n, device=dev) for r, n in zip(st["rows"], st["lens"])])
    page_id, slot = st["table"][seq, pos // st["page"]].long(), pos % st["page"]
    st["k_pages"][page_id, :, slot] = _plain_rotate(st["k"], st["k_norm"], pos).to(st["cache_type"])
    st["v_pages"][page_id, :, slot] = st["v"].to(st["cache_type"])
    return [_plain_rotate(st["q"], st["q_norm"], pos).to(st["cache_type"]), st["k_pages"], st["v_pages"]]


def _plain_attention(st):
    kv, page, heads = st["kv_heads"], st["page"], st["heads"]
    group, first, outs = heads // kv, 0, []
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        q = st["q"][first:first + rows].float().view(rows, kv, group, HEAD_DIM).permute(1, 2, 0, 3)
        first += rows
        if length == 0:
            outs.append(torch.zeros((rows, heads, HEAD_DIM), device=q.device))
            continue
        ids = st["table"][s, :(length + page - 1) // page].long()
        k = st["k_pages"][ids].permute(1, 0, 2, 3).reshape(kv, 1, -1, HEAD_DIM)[:, :, :length].float()
        v = st["v_pages"][ids].permute(1, 0, 2, 3).reshape(kv, 1, -1, HEAD_DIM)[:, :, :length].float()
        step = max(1, (1 << 29) // (heads * length))            # at most 2 GB of scores at a time
        for a in range(0, rows, step):
            b = min(rows, a + step)
            pos = torch.arange(length - rows + a, length - rows + b, device=q.device)
            score = torch.matmul(q[:, :, a:b], k.transpose(-1, -2)) * (1.0 / math.sqrt(HEAD_DIM))
            score = score.masked_fill(torch.arange(length, device=q.device) > pos[:, None], -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            outs.append(o.permute(2, 0, 1, 3).reshape(b - a, heads, HEAD_DIM))
    return torch.cat(outs).to(st["out"].dtype)


# ---- the definitions in 64 bits, sequence by sequence and head by head -------------------------

def _exact_turn(x, weight, angle):
    """x [rows][128]: RMSNorm, then the pairs (j, j + 64) turned by angle [rows][64]."""
    x = x.double()
    x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / HEAD_DIM + EPS)
    z = torch.complex(x[:, :64], x[:, 64:]) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([z.real, z.imag], -1)


def _exact_append(st):
    q_out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    freq = torch.tensor([math.exp(-j / 64 * math.log(THETA)) for j in range(64)], dtype=torch.float64,
                        device=q_out.device)
    table, first, page = st["table"].tolist(), 0, st["page"]
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        span = slice(first, first + rows)
        first += rows
        pos = torch.arange(length - rows, length, dtype=torch.float64, device=q_out.device)
        angle = pos[:, None] * freq
        for h in range(st["heads"]):
            q_out[span, h] = _exact_turn(st["q"][span, h], st["q_norm"], angle)
        for h in range(st["kv_heads"]):
            key, value = _exact_turn(st["k"][span, h], st["k_norm"], angle), st["v"][span, h].double()
            p = length - rows
            while p < length:                                    # one run of rows per page
                end = min(length, (p // page + 1) * page)
                at, src = slice(p % page, p % page + end - p), slice(p - (length - rows), end - (length - rows))
                k_pages[table[s][p // page], h, at] = key[src]
                v_pages[table[s][p // page], h, at] = value[src]
                p = end
    return [q_out, k_pages, v_pages]


def _exact_attention(st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    group, first, page = st["heads"] // st["kv_heads"], 0, st["page"]
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        base = first
        first += rows
        pages = st["table"][s, :(length + page - 1) // page].tolist()
        for h in range(st["kv_heads"] if length else 0):
            key = torch.cat([st["k_pages"][p, h] for p in pages])[:length].double()
            value = torch.cat([st["v_pages"][p, h] for p in pages])[:length].double()
            for a in range(0, rows, 1024):
                b = min(rows, a + 1024)
                seen = length - rows + b                         # keys the block's last row sees
                q = st["q"][base + a:base + b, h * group:(h + 1) * group].double()
                t = torch.einsum("rgd,kd->grk", q, key[:seen]) / HEAD_DIM ** 0.5
                last = torch.arange(seen - (b - a), seen, device=t.device)[:, None]
                t = torch.where(torch.arange(seen, device=t.device) <= last, t, torch.full_like(t, -math.inf))
                w = torch.exp(t - torch.logsumexp(t, -1, keepdim=True))
                out[base + a:base + b, h * group:(h + 1) * group] = torch.einsum("grk,kd->rgd", w, value[:seen])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_append(st) if case["op"] == "append" else _exact_attention(st)
