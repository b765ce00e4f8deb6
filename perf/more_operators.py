"""Serving operators on the paged key-value cache with fewer bytes to a position and to a batch: what is measured,
their plain forms and their definitions in 64 bits.

  append  QK-norm and rotation (both layouts, part of the head, scaled for long contexts) of packed rows; keys and values
          into the cache.  A Q8_0 cache (int8 codes, one f32 scale to 64 elements) quantises them as they are written,
          and the rows are read back as the bf16 values of what it holds; an f32 or bf16 cache is returned as it is.
  read    the rows of sequences read back from the cache, dense
  decode  attention of one new token per sequence over a Q8_0 cache
  prompt  causal attention of packed prompt rows over a Q8_0 cache
  shared  attention of one new token per sequence where groups of sequences share their first pages, which are attended
          to once for the whole group

A case holds sizes only; `layout` derives the ragged lengths from them.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
GROUP = 64
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# theta, rotated elements of a head, layout, and the scaling for contexts longer than the trained ones
ROPES = {
    "plain": dict(theta=1e6, dim=128, interleaved=False, scaling=None, factor=1.0, original=0),
    "yarn": dict(theta=1e6, dim=128, interleaved=False, scaling="yarn", factor=4.0, original=32768),
    "linear": dict(theta=1e6, dim=128, interleaved=False, scaling="linear", factor=8.0, original=0),
    "pairs": dict(theta=1e4, dim=128, interleaved=True, scaling=None, factor=1.0, original=0),
    "part_pairs": dict(theta=1e4, dim=64, interleaved=True, scaling=None, factor=1.0, original=0),
    "part": dict(theta=1e6, dim=96, interleaved=False, scaling="yarn", factor=2.5, original=4096),
}
BETA_FAST, BETA_SLOW = 32.0, 1.0
_handle = None


def listed():
    return [
        # one sequence's next token far out in a context four times the trained one: all latency
        dict(name="append_token", op="append", seqs=1, rows=1, prefix=100002, heads=32, kv_heads=8, page=64,
             io="f32", cache="q8", rope="yarn", mix=1),
        # a packed prefill batch of 4096 tokens into a quantised cache
        dict(name="append_prefill", op="append", seqs=6, rows=4096, prefix=0, heads=32, kv_heads=8, page=64,
             io="f32", cache="q8", rope="plain", mix=2),
        # ragged chunks, half of each head turned in neighbouring pairs, a bf16 cache
        dict(name="append_part", op="append", seqs=5, rows=2001, prefix=8192, heads=16, kv_heads=8, page=16,
             io="bf16", cache="bf16", rope="part_pairs", mix=3),
        # a short sequence's cache handed over as f32 rows
        dict(name="read_one", op="read", seqs=1, longest=300, heads=16, kv_heads=8, page=16, io="f32", cache="q8", mix=4),
        # a batch of cached prompts moved out as bf16
        dict(name="read_batch", op="read", seqs=8, longest=8192, heads=32, kv_heads=8, page=64, io="bf16", cache="q8",
             mix=5),
        # single-user decoding behind 511 positions
        dict(name="decode_one", op="decode", seqs=1, longest=512, heads=16, kv_heads=8, page=16, io="f32", cache="q8",
             mix=6),
        # a full serving batch, lengths spread over 0..16384
        dict(name="decode_batch", op="decode", seqs=64, longest=16384, heads=32, kv_heads=8, page=64, io="bf16",
             cache="q8", mix=7),
        # a packed prefill batch of 4096 tokens in six prompts
        dict(name="prompt_packed", op="prompt", seqs=6, rows=4096, prefix=0, heads=32, kv_heads=8, page=64, io="bf16",
             cache="q8", mix=8),
        # ragged chunks behind long cached prefixes (chunked prefill)
        dict(name="prompt_chunk", op="prompt", seqs=4, rows=2043, prefix=8192, heads=32, kv_heads=8, page=64, io="bf16",
             cache="q8", mix=9),
        # five continuations of one short conversation
        dict(name="shared_few", op="shared", groups=1, seqs=5, prefix=700, tail=90, heads=16, kv_heads=8, page=16,
             io="bf16", cache="bf16", mix=10),
        # a serving batch behind one long system prompt
        dict(name="shared_batch", op="shared", groups=1, seqs=64, prefix=16384, tail=512, heads=32, kv_heads=8, page=64,
             io="bf16", cache="bf16", mix=11),
        # a larger batch behind three of them, the cache quantised
        dict(name="shared_groups", op="shared", groups=3, seqs=150, prefix=12001, tail=1024, heads=40, kv_heads=8,
             page=128, io="bf16", cache="q8", mix=12),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "decode", "prompt", "shared", "shared"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (40, 8), (8, 8), (64, 8), (12, 4), (16, 1)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]), io=rng.choice(["f32", "bf16"]),
                cache="q8", mix=rng.randrange(1, 1 << 20))
    if op == "append":
        case["cache"] = rng.choice(["q8", "q8", "bf16", "f32"])
        case["rope"] = rng.choice(sorted(ROPES))
        case["rows"] = _spread(rng, 1, 4096)
        case["seqs"] = _spread(rng, 1, min(64, case["rows"]))
        case["prefix"] = rng.choice([0, _spread(rng, 1, 100000)])
    elif op in ("read", "decode"):
        case["cache"] = rng.choice(["q8", "q8", "bf16"]) if op == "read" else "q8"
        case["seqs"] = _spread(rng, 1, 64 if op == "read" else 128)
        case["longest"] = _spread(rng, 1, min(65536, (1 << (16 if op == "read" else 19)) // case["seqs"]))
    elif op == "prompt":
        case["io"] = "bf16"
        case["rows"] = _spread(rng, 1, 4096)
        case["seqs"] = _spread(rng, 1, min(64, case["rows"]))
        case["prefix"] = rng.choice([0, 0, _spread(rng, 1, 8192)])
        while work(case)["flops"] > 1.7e11:       # long chunks of many heads: behind less, and shorter
            case["rows"], case["prefix"] = case["rows"] - case["rows"] // 4, case["prefix"] // 2
            case["seqs"] = min(case["seqs"], case["rows"])
    else:
        case["io"], case["cache"] = "bf16", rng.choice(["q8", "bf16"])
        case["seqs"] = _spread(rng, 2, 128)
        case["groups"] = rng.randint(1, min(4, case["seqs"]))
        case["prefix"] = _spread(rng, 16, 12000)
        case["tail"] = _spread(rng, 1, 1024)
    return case


def layout(case):
    """(query rows, cache length with them, positions shared) of each sequence, and the sequences of each group."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    if case["op"] == "shared":
        cuts = sorted(rng.sample(range(1, n), case["groups"] - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [n])]
        prefix = [case["prefix"]] + [rng.randint(max(1, case["prefix"] // 2), case["prefix"]) for _ in sizes[1:]]
        shared = [p for p, size in zip(prefix, sizes) for _ in range(size)]
        return [1] * n, [p + rng.randint(1, case["tail"]) for p in shared], shared, sizes
    if case["op"] in ("decode", "read"):
        lens = [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(n - 1)]
        if n > 4:
            lens[n // 2] = 0                      # an empty slot of the batch
        return (lens if case["op"] == "read" else [1] * n), lens, [0] * n, []
    cuts = sorted(rng.sample(range(1, case["rows"]), n - 1)) if n > 1 else []
    rows = [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]
    prefix = [case["prefix"]] + [rng.randint(0, case["prefix"]) for _ in range(n - 1)]
    return rows, [p + r for p, r in zip(prefix, rows)], [0] * n, []


def work(case):
    rows, lens, shared, sizes = layout(case)
    io = {"f32": 4, "bf16": 2}[case["io"]]
    side = HEAD_DIM + 4 * HEAD_DIM // GROUP if case["cache"] == "q8" else HEAD_DIM * {"f32": 4, "bf16": 2}[case["cache"]]
    total, heads, kv = sum(rows), case["heads"], case["kv_heads"]
    q_out = 4 if case["cache"] == "f32" else 2
    if case["op"] == "append":
        moved = total * (heads + 2 * kv) * HEAD_DIM * io + total * heads * HEAD_DIM * q_out + total * 2 * kv * side
        if case["cache"] == "q8":                 # and read back
            moved += total * 2 * kv * (side + HEAD_DIM * 2)
        # per query or key element: square and sum, scale and weight, half a rotation
        return {"bytes": moved, "flops": total * (heads + kv) * HEAD_DIM * 7}
    if case["op"] == "read":
        return {"bytes": total * 2 * kv * (side + HEAD_DIM * io), "flops": total * 2 * kv * HEAD_DIM}
    if case["op"] == "prompt":
        pairs = sum(r * n - r * (r - 1) // 2 for r, n in zip(rows, lens))
    else:
        pairs = sum(lens)
    keys = sum(lens)
    if sizes:                                     # a group's shared positions once
        first = 0
        for size in sizes:
            keys -= (size - 1) * shared[first]
            first += size
    return {"bytes": 2 * total * heads * HEAD_DIM * io + 2 * keys * kv * side, "flops": 4 * HEAD_DIM * heads * pairs}


def _quantise(x):
    """Q8_0 codes and scales of the last dimension's groups of 64."""
    x = x.unflatten(-1, (-1, GROUP))
    scale = x.abs().amax(-1) / 127.0
    code = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x))
    return torch.trunc(code + torch.copysign(torch.full_like(code, 0.5), code)).flatten(-2), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, lens, shared, sizes = layout(case)
    n, page, heads, kv = len(rows), case["page"], case["heads"], case["kv_heads"]
    total, io, op, q8 = sum(rows), TYPES[case["io"]], case["op"], case["cache"] == "q8"

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    # the table: pages in no order; an append touches the pages of its own rows only (its earlier pages are all page
    # 0), a group's later sequences have the first one's pages as far as all of a page is shared
    max_pages = max(1, max((length + page - 1) // page for length in lens))
    table, need = torch.full((n, max_pages), -1, dtype=torch.int32), []
    first = [(length - r) // page if op == "append" else 0 for r, length in zip(rows, lens)]
    lead, at = {}, 0
    for size in sizes:
        lead.update({s: at for s in range(at + 1, at + size)})
        at += size
    for s, length in enumerate(lens):
        if s in lead:
            first[s] = shared[s] // page
        need.append((length + page - 1) // page - first[s])
    ids = list(range(1, 1 + sum(need)))
    random.Random(seed).shuffle(ids)
    copies = []                                   # pages that are shared in part: (from, to)
    for s in range(n):
        mine = torch.tensor(ids[:need[s]], dtype=torch.int32)
        del ids[:need[s]]
        table[s, :first[s]] = table[lead[s], :first[s]] if s in lead else 0
        table[s, first[s]:first[s] + need[s]] = mine
        if s in lead and shared[s] % page:
            copies.append((int(table[lead[s], first[s]]), int(mine[0])))
    n_pages = 1 + sum(need)

    def pool():
        codes = torch.empty((n_pages, kv, page, HEAD_DIM), dtype=torch.int8 if q8 else TYPES[case["cache"]], device=dev)
        scales = torch.empty((n_pages, kv, page, HEAD_DIM // GROUP), device=dev) if q8 else None
        for a in range(0, n_pages, 4096):
            x = normal(min(4096, n_pages - a), kv, page, HEAD_DIM)
            if q8:
                code, scales[a:a + 4096] = _quantise(x)
                codes[a:a + 4096] = code.to(torch.int8)
            else:
                codes[a:a + 4096] = x
        for t in (codes, scales):
            if copies and t is not None:
                src, dst = (torch.tensor(x, device=dev) for x in zip(*copies))
                t[dst] = t[src]
        return codes, scales

    st = dict(op=op, rows=rows, lens=lens, heads=heads, kv_heads=kv, page=page, q8=q8, io=io, table=table.to(dev),
              kv_len=torch.tensor(lens, dtype=torch.int32, device=dev), shared=shared, sizes=sizes,
              row_off=torch.tensor([0] + rows, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev))
    (st["k_pages"], st["k_scale"]), (st["v_pages"], st["v_scale"]) = pool(), pool()
    if op == "append":
        # the rows of the fused Q|K|V projection, a few channels of it large
        qkv = normal(total, heads + 2 * kv, HEAD_DIM)
        qkv[:, :, 5::50] *= 6.0
        qkv = qkv.to(io)
        q_type = torch.float32 if case["cache"] == "f32" else torch.bfloat16
        st.update(q=qkv[:, :heads], k=qkv[:, heads:heads + kv], v=qkv[:, heads + kv:], rope=ROPES[case["rope"]],
                  q_norm=1 + 0.2 * normal(HEAD_DIM), k_norm=1 + 0.2 * normal(HEAD_DIM),
                  out=torch.empty((total, heads, HEAD_DIM), dtype=q_type, device=dev))
    elif op != "read":
        # normalised queries with a little gain, so that the softmax is neither flat nor a single key
        q = normal(total, heads, HEAD_DIM)
        q = 1.5 * q * torch.rsqrt((q * q).mean(-1, keepdim=True))
        st.update(q=q.to(io), out=torch.empty((total, heads, HEAD_DIM), dtype=io, device=dev))
    if op == "read" or (op == "append" and q8):
        st["back"] = [torch.empty((total, kv, HEAD_DIM), dtype=io if op == "read" else torch.bfloat16, device=dev)
                      for _ in range(2)]
    if own:
        global _handle
        from metalqwen3_b200.q3cu import KVBatch, KVCache, KVPrefix, Q3CU, Rope
        if _handle is None:
            _handle = Q3CU(0)
        st["q3"] = _handle
        st["cache"] = KVCache(st["k_pages"], st["v_pages"], st["k_scale"], st["v_scale"])
        st["batch"] = KVBatch(st["kv_len"], st["table"], st["row_off"])
        if op == "append":
            st["turn"] = Rope(**st["rope"], beta_fast=BETA_FAST, beta_slow=BETA_SLOW)
        if op == "decode":
            st["space"] = _handle.attention_paged_workspace(st["cache"], heads)
        if op == "shared":
            off = torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0, dtype=torch.int32)
            length = torch.tensor([shared[a] for a in off[:-1].tolist()], dtype=torch.int32)
            st["prefix"] = KVPrefix(off.to(dev), length.to(dev))
            st["space"] = _handle.attention_shared_workspace(st["cache"], n, heads)
    return st


def run(st):
    if own:
        q3, cache, batch = st["q3"], st["cache"], st["batch"]
        if st["op"] == "append":
            q = q3.kv_append(cache, batch, st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"], eps=EPS,
                             rope=st["turn"], q_out=st["out"])
            if not st["q8"]:
                return [q, st["k_pages"], st["v_pages"]]
            return [q, *q3.kv_read(cache, batch, k_out=st["back"][0], v_out=st["back"][1])]
        if st["op"] == "read":
            return list(q3.kv_read(cache, batch, k_out=st["back"][0], v_out=st["back"][1]))
        if st["op"] == "decode":
            return q3.attention_paged(cache, batch, st["q"], out=st["out"], work=st["space"])
        if st["op"] == "shared":
            return q3.attention_shared(cache, batch, st["prefix"], st["q"], out=st["out"], work=st["space"])
        return q3.attention_prompt(cache, batch, st["q"], out=st["out"])
    if st["op"] == "append":
        return _plain_append(st)
    return _plain_read(st, st["io"]) if st["op"] == "read" else _plain_attention(st)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ------------------

def _plain_frequencies(rope, device):
    """Radians a position of each rotated pair (64 bits), and the factor of cosine and sine."""
    half, theta, factor = rope["dim"] // 2, rope["theta"], rope["factor"]
    j = torch.arange(half, dtype=torch.float64, device=device)
    freq = theta ** (-j / half)
    if rope["scaling"] == "linear":
        return freq / factor, 1.0
    if rope["scaling"] == "yarn":
        # pairs that turn more than BETA_FAST times over the trained length keep their frequency, those that turn less
        # than BETA_SLOW times are slowed by the factor, with a ramp over the pairs between
        def pair(turns):
            return rope["dim"] * math.log(rope["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(BETA_FAST)), 0), min(math.ceil(pair(BETA_SLOW)), rope["dim"] - 1)
        ramp = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
        return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _plain_rotate(x, weight, pos, rope, dtype):
    # (what is quantised next in 64 bits: it may lie next to the border of two codes)
    x = x.to(dtype)
    x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * weight
    freq, factor = _plain_frequencies(rope, x.device)
    angle = pos.double()[:, None, None] * freq       # 64 bits: positions reach far past a turn's precision in 32
    c, s = (torch.cos(angle) * factor).to(x.dtype), (torch.sin(angle) * factor).to(x.dtype)
    turned, rest = x[..., :rope["dim"]], x[..., rope["dim"]:]
    if rope["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, rest], -1)


def _slots(st):
    """Sequence, page and slot of every packed row, and the rows' positions."""
    dev = st["table"].device
    seq = torch.cat([torch.full((r,), s, dtype=torch.long, device=dev) for s, r in enumerate(st["rows"])])
    pos = torch.cat([torch.arange(n - r, n, device=dev) for r, n in zip(st["rows"], st["lens"])])
    return st["table"][seq, pos // st["page"]].long(), pos % st["page"], pos


def _plain_append(st):
    page_id, slot, pos = _slots(st)
    wide = torch.float64 if st["q8"] else torch.float32
    key, value = _plain_rotate(st["k"], st["k_norm"], pos, st["rope"], wide), st["v"].to(wide)
    q = _plain_rotate(st["q"], st["q_norm"], pos, st["rope"], torch.float32).to(st["out"].dtype)
    for pages, scales, x in ((st["k_pages"], st["k_scale"], key), (st["v_pages"], st["v_scale"], value)):
        if st["q8"]:
            code, scale = _quantise(x)
            pages[page_id, :, slot], scales[page_id, :, slot] = code.to(torch.int8), scale.float()
        else:
            pages[page_id, :, slot] = x.to(pages.dtype)
    return [q] + (_plain_read(st, torch.bfloat16) if st["q8"] else [st["k_pages"], st["v_pages"]])


def _values(st, side, page_id, slot):
    """What the cache holds at (page, slot), [rows][kv heads][128] in 32 bits."""
    x = st[side + "_pages"][page_id, :, slot].float()
    return x * st[side + "_scale"][page_id, :, slot].repeat_interleave(GROUP, -1) if st["q8"] else x


def _plain_read(st, dtype):
    page_id, slot, _ = _slots(st)
    return [_values(st, side, page_id, slot).to(dtype) for side in "kv"]


def _plain_attention(st):
    kv, page, heads = st["kv_heads"], st["page"], st["heads"]
    group, first, outs = heads // kv, 0, []
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        q = st["q"][first:first + rows].float().view(rows, kv, group, HEAD_DIM).permute(1, 2, 0, 3)
        first += rows
        if length == 0:
            outs.append(torch.zeros((rows, heads, HEAD_DIM), device=q.device))
            continue
        at = torch.arange(length, device=q.device)
        page_id, slot = st["table"][s, at // page].long(), at % page
        k, v = (_values(st, side, page_id, slot).permute(1, 0, 2)[:, None] for side in "kv")
        step = max(1, (1 << 29) // (heads * length))            # at most 2 GB of scores at a time
        for a in range(0, rows, step):
            b = min(rows, a + step)
            pos = torch.arange(length - rows + a, length - rows + b, device=q.device)
            score = torch.matmul(q[:, :, a:b], k.transpose(-1, -2)) * (1.0 / math.sqrt(HEAD_DIM))
            score = score.masked_fill(at > pos[:, None], -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            outs.append(o.permute(2, 0, 1, 3).reshape(b - a, heads, HEAD_DIM))
    return torch.cat(outs).to(st["out"].dtype)


# ---- the definitions in 64 bits, sequence by sequence and head by head -------------------------

def _exact_turns(rope, device):
    """exp(i a) a position's worth of each pair as angles, from the scaling's definition pair by pair."""
    angles, d = [], rope["dim"]
    for j in range(d // 2):
        f = math.exp(-2.0 * j / d * math.log(rope["theta"]))
        if rope["scaling"] == "linear":
            f /= rope["factor"]
        elif rope["scaling"] == "yarn":
            edge = [d / (2.0 * math.log(rope["theta"])) * math.log(rope["original"] / (2.0 * math.pi * b))
                    for b in (BETA_FAST, BETA_SLOW)]
            lo, hi = max(0, math.floor(edge[0])), min(d - 1, math.ceil(edge[1]))
            share = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            f = f / rope["factor"] * share + f * (1.0 - share)
        angles.append(f)
    gain = 1.0 + 0.1 * math.log(rope["factor"]) if rope["scaling"] == "yarn" else 1.0
    return torch.tensor(angles, dtype=torch.float64, device=device), gain


def _exact_turn(x, weight, pos, turns, rope):
    """x [rows][128]: RMSNorm, then the pairs turned as complex numbers."""
    x = x.double()
    x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / HEAD_DIM + EPS)
    d, (freq, gain) = rope["dim"], turns
    angle = pos.double()[:, None] * freq
    pairs = x[:, :d].unflatten(-1, (-1, 2)).transpose(-1, -2) if rope["interleaved"] else x[:, :d].unflatten(-1, (2, -1))
    z = torch.complex(pairs[:, 0], pairs[:, 1]) * torch.polar(torch.full_like(angle, gain), angle)
    both = torch.stack([z.real, z.imag], 1)
    x[:, :d] = (both.transpose(-1, -2) if rope["interleaved"] else both).flatten(-2)
    return x


def _exact_held(x):
    """What a Q8_0 cache holds of rows x (64 bits): the nearest whole multiple, half away from zero, of each group's step."""
    out = torch.zeros_like(x)
    for g in range(0, HEAD_DIM, GROUP):
        part = x[..., g:g + GROUP]
        step = part.abs().amax(-1, keepdim=True) / 127.0
        whole = (part.abs() / step.clamp_min(1e-300) + 0.5).floor()
        out[..., g:g + GROUP] = part.sign() * whole * step
    return out


def _exact_append(st):
    dev = st["q"].device
    q_out = torch.empty(st["q"].shape, dtype=torch.float64, device=dev)
    if st["q8"]:
        back = [torch.empty(st["k"].shape, dtype=torch.float64, device=dev) for _ in range(2)]
    else:
        k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    turns = _exact_turns(st["rope"], dev)
    table, first, page = st["table"].tolist(), 0, st["page"]
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        span = slice(first, first + rows)
        first += rows
        pos = torch.arange(length - rows, length, device=dev)
        for h in range(st["heads"]):
            q_out[span, h] = _exact_turn(st["q"][span, h], st["q_norm"], pos, turns, st["rope"])
        for h in range(st["kv_heads"]):
            key = _exact_turn(st["k"][span, h], st["k_norm"], pos, turns, st["rope"])
            value = st["v"][span, h].double()
            if st["q8"]:
                back[0][span, h], back[1][span, h] = _exact_held(key), _exact_held(value)
                continue
            p = length - rows
            while p < length:                                    # one run of rows per page
                end = min(length, (p // page + 1) * page)
                at, src = slice(p % page, p % page + end - p), slice(p - (length - rows), end - (length - rows))
                k_pages[table[s][p // page], h, at] = key[src]
                v_pages[table[s][p // page], h, at] = value[src]
                p = end
    return [q_out] + (back if st["q8"] else [k_pages, v_pages])


def _exact_side(st, side, pages, h, length):
    """Positions 0 .. length - 1 of kv head h on these pages, in 64 bits."""
    x = torch.cat([st[side + "_pages"][p, h] for p in pages])[:length].double()
    if st["q8"]:
        scale = torch.cat([st[side + "_scale"][p, h] for p in pages])[:length].double()
        x = (x.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)
    return x


def _exact_read(st):
    first, page = 0, st["page"]
    out = [torch.empty(st["back"][0].shape, dtype=torch.float64, device=st["table"].device) for _ in range(2)]
    for s, length in enumerate(st["lens"]):
        pages = st["table"][s, :(length + page - 1) // page].tolist()
        for h in range(st["kv_heads"] if length else 0):
            for side, o in zip("kv", out):
                o[first:first + length, h] = _exact_side(st, side, pages, h, length)
        first += length
    return out


def _exact_attention(st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    group, first, page = st["heads"] // st["kv_heads"], 0, st["page"]
    for s, (rows, length) in enumerate(zip(st["rows"], st["lens"])):
        base = first
        first += rows
        pages = st["table"][s, :(length + page - 1) // page].tolist()
        for h in range(st["kv_heads"] if length else 0):
            key, value = (_exact_side(st, side, pages, h, length) for side in "kv")
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
    if st["op"] == "append":
        return _exact_append(st)
    return _exact_read(st) if st["op"] == "read" else _exact_attention(st)
