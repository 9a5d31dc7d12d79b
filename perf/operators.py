"""Cases that measure the paged 8-bit decode operators: the step plan, the rotary append, attention and gather over the 8-bit
cache, and batched sampling. `own` selects the framework's kernels; otherwise `run` computes the same operators from elementary
torch operations.

Every state is made from a seed: request lengths, a shuffled page assignment (pages of a request are scattered, as after some
time of serving), activations and logits with the spread that a decoder layer and an LM head produce.
"""

from __future__ import annotations

import math
import random

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
LOG2E = 1.4426950408889634
# Taylor coefficients of 2^g, highest power first
EXP2 = [math.log(2.0) ** i / math.factorial(i) for i in range(7, -1, -1)]


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of a busy server: every row grows by a token
        dict(name="plan_decode", op="plan", rows=64, page=64, longest=8192, chunk=1, release=0, room=64),
        # continuous batching: decoding rows, prompt pieces and finished rows in one step, small pages
        dict(name="plan_mixed", op="plan", rows=509, page=16, longest=16384, chunk=2048, release=1, room=131072),
        # K / V of one new token a row, written into open blocks
        dict(name="append_decode", op="append", rows=64, heads=28, kv_heads=4, dim=128, page=64, kv="e4m3", tokens=64,
             dtype="float32"),
        # prompt pieces of a few requests, odd lengths
        dict(name="append_prompt", op="append", rows=5, heads=32, kv_heads=8, dim=128, page=64, kv="e4m3", tokens=16381,
             dtype="bfloat16"),
        # a single user's decode step: latency
        dict(name="attn_one", op="attn", rows=1, heads=32, kv_heads=8, dim=64, page=64, kv="e4m3", longest=4097, q=1),
        # a batch of chats, ragged, some rows empty
        dict(name="attn_batch", op="attn", rows=33, heads=32, kv_heads=8, dim=128, page=64, kv="e4m3", longest=8192, q=1),
        # one long document, int8, few KV heads
        dict(name="attn_long", op="attn", rows=1, heads=16, kv_heads=2, dim=128, page=128, kv="int8", longest=131071, q=1),
        # several tokens a row (drafts to verify), causal among themselves; the largest cache
        dict(name="attn_verify", op="attn", rows=64, heads=28, kv_heads=4, dim=128, page=32, kv="e4m3", longest=32768, q=5),
        # a short session read back before its next segment's prefill
        dict(name="gather_short", op="gather", kv_heads=2, dim=64, page=16, kv="int8", longest=2041),
        # a long one
        dict(name="gather_long", op="gather", kv_heads=8, dim=128, page=64, kv="e4m3", longest=131072),
        # one user's next token
        dict(name="sample_one", op="sample", rows=1, vocab=128256, dtype="float32"),
        # a batch, each row with its own settings
        dict(name="sample_batch", op="sample", rows=129, vocab=151936, dtype="float32"),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["plan", "append", "attn", "attn", "gather", "sample"])
    kv = rng.choice(["e4m3", "int8"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        chunk = rng.choice([1, 4, 256, 2048])
        rows = _log_int(rng, 1, 509)
        return dict(op=op, rows=rows, page=page, longest=_log_int(rng, 64, 16384), chunk=chunk,
                    release=rng.randrange(2), room=rows * chunk if rows * chunk < 4096 else 131072)
    if op == "append":
        rows = _log_int(rng, 1, 128)
        heads, kv_heads, dim = rng.choice([(28, 4, 128), (32, 8, 128), (16, 2, 128), (14, 2, 64), (8, 8, 64)])
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kv=kv,
                    tokens=max(rows, _log_int(rng, 1, 16381)), dtype=rng.choice(["float32", "bfloat16", "float16"]))
    if op == "attn":
        heads, kv_heads, dim = rng.choice([(28, 4, 128), (32, 8, 128), (16, 2, 128), (14, 2, 64), (32, 8, 64), (8, 8, 128)])
        rows = _log_int(rng, 1, 64)
        most = 64 * 32768 * 4 * 128 // (rows * kv_heads * dim)
        q = rng.choice([1, 1, 1, 2, 5])
        return dict(op=op, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kv=kv,
                    longest=_log_int(rng, 16, max(16, min(most, 131072))), q=q)
    if op == "gather":
        kv_heads, dim = rng.choice([(8, 128), (4, 128), (2, 128), (2, 64), (8, 64)])
        return dict(op=op, kv_heads=kv_heads, dim=dim, page=page, kv=kv, longest=_log_int(rng, 1000, 131072))
    return dict(op=op, rows=_log_int(rng, 1, 129), vocab=_log_int(rng, 1000, 151936),
                dtype=rng.choice(["float32", "bfloat16"]))


# --------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Request lengths, log-uniform up to `longest`, the first one the longest, every eleventh row empty."""
    r = random.Random(seed * 7919 + 13)
    out = []
    for i in range(case["rows"]):
        if i == 0:
            out.append(case["longest"])
        elif i % 11 == 10:
            out.append(0)
        else:
            out.append(_log_int(r, max(1, case["longest"] // 16), case["longest"]))
    return out


def _tables(lengths, page, g, dev, pages=None, width=None):
    """Block tables with scattered pages for `lengths`, and the free pages of the pool."""
    have = [-(-n // page) for n in lengths]
    pages = pages or sum(have) + 8
    width = width or max(have) + 1
    order = torch.randperm(pages, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    col = torch.arange(width, device=dev).unsqueeze(0)
    held = torch.tensor(have, device=dev).unsqueeze(1)
    first = torch.cumsum(held, 0) - held
    at = (first + col).clamp(max=pages - 1)
    table = torch.where(col < held, order[at], torch.full_like(order[at], -1))
    return table.contiguous(), order[sum(have):].contiguous(), pages


def _pool(pages, case, g, dev, which):
    """One cache tensor [pages, kv_heads, page, dim] in 8 bits and its scales [pages, kv_heads] (powers of two, as the append
    makes them): values of unit spread, some heads larger."""
    kvh, page, dim = case["kv_heads"], case["page"], case["dim"]
    spread = 2.0 ** torch.randint(-1, 2, (pages, kvh), generator=g, device=dev).float()
    if case["kv"] == "e4m3":
        scale = spread * 2.0 ** (-6 if which == "k" else -7)
        data = torch.empty(pages, kvh, page, dim, device=dev, dtype=torch.float8_e4m3fn)
    else:
        scale = spread * 2.0 ** -5
        data = torch.empty(pages, kvh, page, dim, device=dev, dtype=torch.int8)
    amp = 60.0 if case["kv"] == "e4m3" else 30.0
    step = max(1, (1 << 27) // (kvh * page * dim))
    at = 0
    while at < pages:
        n = min(step, pages - at)
        x = torch.randn(n, kvh, page, dim, generator=g, device=dev) * amp
        if case["kv"] == "e4m3":
            data[at:at + n] = x.clamp(-448, 448).to(torch.float8_e4m3fn)
        else:
            data[at:at + n] = x.round().clamp(-127, 127).to(torch.int8)
        at += n
    return data, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"op": case["op"], "case": case}
    if case["op"] == "plan":
        r = random.Random(seed)
        lens = _lengths(case, seed)
        add, left = [], case["room"] - case["rows"]
        for i in range(case["rows"]):
            if case["release"] and i % 7 == 5:
                add.append(-1)
            elif case["chunk"] > 1 and i % 4 == 1:
                n = min(left, _log_int(r, 1, case["chunk"]))
                left -= n
                add.append(n)
            else:
                add.append(1)
        width = (case["longest"] + case["chunk"]) // case["page"] + 2
        table, free, pages = _tables(lens, case["page"], g, dev, pages=case["rows"] * width, width=width)
        ring = torch.full((pages,), -1, device=dev, dtype=torch.int32)
        tail = int(free.numel())
        # the ring's counters only grow: a server that has run for a while starts anywhere in it
        head = r.randrange(0, 1 << 20)
        ring[(torch.arange(tail, device=dev) + head) % pages] = free
        s.update(add=torch.tensor(add, device=dev, dtype=torch.int32), kv_len=torch.tensor(lens, device=dev, dtype=torch.int32),
                 table=table, ring=ring, counters=torch.tensor([head, head + tail], device=dev, dtype=torch.int64),
                 page=case["page"], room=case["room"])
        # the buffers that a step's plan lives in, kept by the serving loop
        R, T = case["rows"], case["room"]
        i32 = dict(device=dev, dtype=torch.int32)
        s["out"] = dict(cu=torch.empty(R + 1, **i32), row=torch.empty(T, **i32), pos=torch.empty(T, **i32),
                        slot=torch.empty(T, device=dev, dtype=torch.int64),
                        unit=torch.empty(min(T, T // case["page"] + 2 * R), 4, **i32), kv_len=torch.empty(R, **i32),
                        counters=torch.empty(2, device=dev, dtype=torch.int64), info=torch.empty(4, **i32))
        return s
    if case["op"] == "append":
        H, Hkv, D, P, T, R = (case[k] for k in ("heads", "kv_heads", "dim", "page", "tokens", "rows"))
        r = random.Random(seed)
        cuts = sorted(r.sample(range(1, T), R - 1)) if R > 1 else []
        n = [b - a for a, b in zip([0] + cuts, cuts + [T])]
        old = [r.randrange(0, 4 * P) for _ in range(R)]
        table, _, pages = _tables([o + m for o, m in zip(old, n)], P, g, dev, pages=T // P + 6 * R + 8)
        row = torch.repeat_interleave(torch.arange(R, device=dev), torch.tensor(n, device=dev))
        first = torch.cumsum(torch.tensor(n, device=dev), 0) - torch.tensor(n, device=dev)
        pos = torch.arange(T, device=dev) - first[row] + torch.tensor(old, device=dev)[row]
        slot = table[row, pos // P].long() * P + pos % P
        units, t = [], 0
        for i in range(R):
            p, end = old[i], old[i] + n[i]
            while p < end:
                m = min(end, (p // P + 1) * P) - p
                units.append((i, t, m, p))
                t, p = t + m, p + m
        qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g, device=dev)
        qkv *= 2.0 ** torch.randint(-1, 2, (T, 1), generator=g, device=dev).float()
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D))
        f = torch.arange(max(o + m for o, m in zip(old, n)), dtype=torch.float64, device=dev).unsqueeze(1) * inv
        k, ks = _pool(pages, case, g, dev, "k")
        v, vs = _pool(pages, case, g, dev, "v")
        s.update(qkv=qkv.to(getattr(torch, case["dtype"])), cos=f.cos().float(), sin=f.sin().float(), row=row.to(torch.int32),
                 pos=pos.to(torch.int32), slot=slot, units=torch.tensor(units, device=dev, dtype=torch.int32), table=table,
                 k=k, v=v, k_scale=ks, v_scale=vs, q_out=torch.empty(T, H, D, device=dev, dtype=torch.bfloat16),
                 tokens=T)
        return s
    if case["op"] == "attn":
        H, Hkv, D, P, R = (case[k] for k in ("heads", "kv_heads", "dim", "page", "rows"))
        lens = _lengths(case, seed)
        qn = [case["q"] if i % 3 == 0 else 1 + i % case["q"] for i in range(R)]
        lens = [max(n, m) if n else 0 for n, m in zip(lens, qn)]
        table, _, pages = _tables(lens, P, g, dev)
        k, ks = _pool(pages, case, g, dev, "k")
        v, vs = _pool(pages, case, g, dev, "v")
        cu = torch.zeros(R + 1, device=dev, dtype=torch.int32)
        cu[1:] = torch.cumsum(torch.tensor(qn, device=dev), 0).to(torch.int32)
        q = torch.randn(sum(qn), H, D, generator=g, device=dev) * 1.5
        s.update(q=q.to(torch.bfloat16), k=k, v=v, k_scale=ks, v_scale=vs, table=table, cu=cu,
                 kv_len=torch.tensor(lens, device=dev, dtype=torch.int32), longest=max(lens), most=max(qn),
                 scale=1.0 / math.sqrt(D))
        return s
    if case["op"] == "gather":
        lens = [case["longest"]]
        table, _, pages = _tables(lens, case["page"], g, dev)
        k, ks = _pool(pages, case, g, dev, "k")
        v, vs = _pool(pages, case, g, dev, "v")
        s.update(k=k, v=v, k_scale=ks, v_scale=vs, table=table[0].contiguous(), n=case["longest"])
        return s
    R, V = case["rows"], case["vocab"]
    # an LM head's logits: a broad bulk, and a few strong candidates a row
    logits = torch.randn(R, V, generator=g, device=dev) * 2.0
    top = torch.randint(0, V, (R, 24), generator=g, device=dev)
    logits.scatter_add_(1, top, torch.rand(R, 24, generator=g, device=dev) * 12.0)
    r = random.Random(seed)
    modes = [(0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0),
             (0.9, 1000, 1.0, 0.0), (1.5, 64, 0.8, 0.02)]
    pick = [modes[(i + (r.randrange(len(modes)) if R > 1 else 0)) % len(modes)] for i in range(R)]
    col = lambda i, dt: torch.tensor([m[i] for m in pick], device=dev, dtype=dt)  # noqa: E731
    s.update(logits=logits.to(getattr(torch, case["dtype"])), u=torch.rand(R, generator=g, device=dev),
             temperature=col(0, torch.float32), top_k=col(1, torch.int32), top_p=col(2, torch.float32), min_p=col(3, torch.float32))
    return s


# --------------------------------------------------------------------------- the plain forms
def _plan_plain(s):
    add, old, table, ring, P, room = s["add"].long(), s["kv_len"].long(), s["table"], s["ring"], s["page"], s["room"]
    R, W = table.shape
    dev = add.device
    head, tail = s["counters"][0], s["counters"][1]
    gone = add < 0
    n = add.clamp(min=0)
    new = torch.where(gone, 0, old + n)
    have = (old + P - 1) // P
    need = torch.where(gone, 0, (old + n + P - 1) // P - have)
    back = torch.where(gone, have, 0)
    total, popped, pushed = n.sum(), need.sum(), back.sum()
    bad = (popped > tail - head + pushed) | (need + have > W).any() | (total > room)
    status = torch.where(total > room, 3, torch.where((need + have > W).any(), 2, torch.where(bad, 1, 0)))
    n, need, back = n * ~bad, need * ~bad, back * ~bad
    new = torch.where(bad, old, new)
    col = torch.arange(W, device=dev).unsqueeze(0)
    # released pages in row order behind the free ones
    first_back = torch.cumsum(back, 0) - back
    size = ring.numel()
    ring = ring.clone()
    put = col < back.unsqueeze(1)
    at = torch.where(put, (tail + first_back.unsqueeze(1) + col) % size, size)
    pad = torch.cat([ring, ring.new_zeros(1)])
    pad[at.reshape(-1)] = table.reshape(-1)
    ring = pad[:size]
    first_need = torch.cumsum(need, 0) - need
    j = col - have.unsqueeze(1)
    take = (j >= 0) & (j < need.unsqueeze(1))
    table = torch.where(take, ring[(head + first_need.unsqueeze(1) + j) % size], table)
    cu = torch.zeros(R + 1, device=dev, dtype=torch.int64)
    cu[1:] = torch.cumsum(n, 0)
    t = torch.arange(room, device=dev)
    live = t < cu[-1]
    row = torch.searchsorted(cu[1:], t, right=True).clamp(max=R - 1)
    pos = t - cu[row] + old[row]
    slot = table[row, (pos // P).clamp(0, W - 1)].long() * P + pos % P
    units = torch.where(n > 0, (old + n + P - 1) // P - old // P, 0)
    cap = min(room, room // P + 2 * R)
    cun = torch.zeros(R + 1, device=dev, dtype=torch.int64)
    cun[1:] = torch.cumsum(units, 0)
    i = torch.arange(cap, device=dev)
    ur = torch.searchsorted(cun[1:], i, right=True).clamp(max=R - 1)
    block = old[ur] // P + i - cun[ur]
    p0 = torch.maximum(block * P, old[ur])
    p1 = torch.minimum((block + 1) * P, (old + n)[ur])
    unit = torch.stack([ur, cu[ur] + p0 - old[ur], p1 - p0, p0], 1)
    unit = torch.where((i < cun[-1]).unsqueeze(1), unit, torch.tensor([-1, 0, 0, 0], device=dev))
    i32 = torch.int32
    return {"cu": cu.to(i32), "row": torch.where(live, row, -1).to(i32), "pos": torch.where(live, pos, 0).to(i32),
            "slot": torch.where(live, slot, -1), "unit": unit.to(i32), "kv_len": new.to(i32),
            "counters": torch.stack([head + popped * ~bad, tail + pushed * ~bad]),
            "info": torch.stack([total * ~bad, cun[-1], popped * ~bad, status]).to(i32), "table": table, "ring": ring}


def _pow2_scale(amax, kv):
    """The smallest power of two s (2^-40 to 2^40) with amax <= QMAX * s."""
    m, e = torch.frexp(amax)
    lim, sub = (0.875, 9) if kv == "e4m3" else (0.9921875, 7)
    e = torch.where(m <= lim, e - sub, e - sub + 1).clamp(-40, 40)
    e = torch.where(amax > 0, e, -40)
    return torch.ldexp(torch.ones_like(amax), e)


def _to8(x, kv):
    return x.clamp(-448, 448).to(torch.float8_e4m3fn) if kv == "e4m3" else x.round().clamp(-127, 127).to(torch.int8)


def _take(data, *index):
    """data[index] by way of its bytes (8-bit floats have no indexing of their own)."""
    return data.view(torch.uint8)[index].view(data.dtype).float()


def _store_plain(x, data, scale, slot, units, table, P, kv):
    """Rows x [T, heads, D] into their slots; an open block's stored values are rescaled when its scale grows."""
    page, off = slot // P, slot % P
    amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
    upage = table[units[:, 0].long(), units[:, 3].long() // P].long()
    start = (units[:, 3] % P).long()
    old = torch.where((start == 0).unsqueeze(1), 0.0, scale[upage])
    new = torch.maximum(old, _pow2_scale(amax[upage], kv))
    have = _take(data, upage)
    again = _to8(have * (old / new).view(*old.shape, 1, 1), kv)
    keep = (torch.arange(P, device=x.device) < start.unsqueeze(1)).view(-1, 1, P, 1) & (old < new).view(*old.shape, 1, 1)
    raw = data.view(torch.uint8)
    raw[upage] = torch.where(keep, again.view(torch.uint8), raw[upage])
    scale[upage] = new
    raw[page, :, off] = _to8(x / scale[page].unsqueeze(-1), kv).view(torch.uint8)


def _append_plain(s):
    c = s["case"]
    H, Hkv, D, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    T = s["tokens"]
    x = s["qkv"].float().view(T, H + 2 * Hkv, D)
    pos = s["pos"].long()
    cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
    x1, x2 = x[:, :H + Hkv, :D // 2], x[:, :H + Hkv, D // 2:]
    rot = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    _store_plain(rot[:, H:], s["k"], s["k_scale"], s["slot"], s["units"], s["table"], P, c["kv"])
    _store_plain(x[:, H + Hkv:], s["v"], s["v_scale"], s["slot"], s["units"], s["table"], P, c["kv"])
    return rot[:, :H].to(torch.bfloat16)


def _rows_plain(data, scale, table, n, P):
    """The first n cached rows of each table row, [R, n, heads, D] in float32."""
    j = torch.arange(n, device=table.device)
    page = table[..., j // P].clamp(min=0).long()
    return _take(data, page, slice(None), j % P) * scale[page].unsqueeze(-1)


def _attn_plain(s):
    c = s["case"]
    H, Hkv, P, R = c["heads"], c["kv_heads"], c["page"], c["rows"]
    n, m = s["longest"], s["most"]
    k = _rows_plain(s["k"], s["k_scale"], s["table"], n, P)
    cu, lens = s["cu"].long(), s["kv_len"].long()
    qn = cu[1:] - cu[:-1]
    i = torch.arange(m, device=k.device)
    here = i < qn.unsqueeze(1)
    at = (cu[:-1].unsqueeze(1) + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].view(R, m, Hkv, H // Hkv, -1)
    a = torch.einsum("rihgd,rjhd->rhgij", q, k) * s["scale"]
    del k
    limit = (lens - qn).unsqueeze(1) + i
    seen = torch.arange(n, device=a.device).view(1, 1, -1) <= limit.unsqueeze(2)
    a = a.masked_fill(~seen.view(R, 1, 1, m, n), float("-inf"))
    top = a.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(a - top)
    del a
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), float("-inf")).squeeze(-1)
    p /= total.clamp(min=1e-30)
    v = _rows_plain(s["v"], s["v_scale"], s["table"], n, P)
    o = torch.einsum("rhgij,rjhd->rihgd", p, v).reshape(R, m, H, -1)
    return {"o": o[here].to(torch.bfloat16), "lse": lse.permute(0, 3, 1, 2).reshape(R, m, H)[here].t().contiguous()}


def _gather_plain(s):
    P = s["case"]["page"]
    return [_rows_plain(s[x], s[x + "_scale"], s["table"], s["n"], P).permute(1, 0, 2).to(torch.bfloat16).contiguous() for x in "kv"]


def _share(total, x):
    """floor(total * x) for x in [0, 1] held in 24 bits."""
    x = (x * 16777216.0).to(torch.int64).clamp(0, 1 << 24)
    return (total >> 24) * x + (((total & 0xFFFFFF) * x) >> 24)


def _sample_plain(s):
    x, T = s["logits"].float(), s["temperature"].unsqueeze(1)
    V = x.shape[1]
    x = torch.where(torch.isnan(x), float("-inf"), x)
    top = x.amax(1, keepdim=True)
    d = torch.where(x == top, 0.0, (top - x) / torch.where(T > 0, T, 1.0))
    d = torch.where(torch.isnan(d), 64.0, d.clamp(max=64.0))
    # the weight exp(-d) in 31 bits: 2^-n 2^g with n + (-g) = d log2(e)
    y = d * LOG2E
    n = y.round()
    g = n - y
    w = torch.full_like(g, EXP2[0])
    w = w * g + EXP2[1]
    w = w * g + EXP2[2]
    w = w * g + EXP2[3]
    w = w * g + EXP2[4]
    w = w * g + EXP2[5]
    w = w * g + EXP2[6]
    w = w * g + EXP2[7]
    w = (w * 2147483648.0).to(torch.int64) >> n.to(torch.int64).clamp(max=62)
    rank, order = torch.sort(d, dim=1, stable=True)
    ws = w.gather(1, order)
    i = torch.arange(V, device=x.device).unsqueeze(0)
    k = s["top_k"].long().unsqueeze(1)
    ws = torch.where((i < k) | (k <= 0), ws, 0)
    cum = torch.cumsum(ws, 1)
    p = s["top_p"].unsqueeze(1)
    limit = torch.where((p > 0) & (p < 1), _share(cum[:, -1:], p).clamp(min=1), 1 << 62)
    ws = torch.where(cum - ws < limit, ws, 0)
    ws = torch.where(ws >= (s["min_p"].clamp(0, 1).unsqueeze(1) * 2147483648.0).to(torch.int64), ws, 0)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    cum = torch.cumsum(kept, 1)
    u = s["u"].clamp(0, 0.99999994).unsqueeze(1)
    token = torch.searchsorted(cum, _share(cum[:, -1:], u), right=True).squeeze(1)
    token = torch.where(s["temperature"] > 0, token, (x == top).to(torch.int8).argmax(1))
    return torch.where(top.squeeze(1) == float("-inf"), -1, token)


# --------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if not own:
        if op == "plan":
            return _plan_plain(s)
        if op == "append":
            q = _append_plain(s)
            return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        return {"attn": _attn_plain, "gather": _gather_plain, "sample": _sample_plain}[op](s)
    from hetero_cp_ringattn_b200.ops import paged, sampling
    if op == "plan":
        paged.plan_step(s["add"], s["kv_len"], s["table"], s["ring"], s["counters"], page=s["page"], max_tokens=s["room"],
                        out=paged.StepPlan(**s["out"]))
        return {**s["out"], "table": s["table"], "ring": s["ring"]}
    if op == "append":
        c = s["case"]
        q = paged.rope_append_kv8(s["qkv"], s["cos"], s["sin"], s["pos"], s["units"], s["table"], s["k"], s["v"], s["k_scale"],
                                  s["v_scale"], heads=c["heads"], q_out=s["q_out"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "attn":
        o, lse = paged.attention_kv8(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["kv_len"],
                                     None if s["most"] == 1 else s["cu"], max_q=s["most"], scale=s["scale"])
        return {"o": o, "lse": lse}
    if op == "gather":
        return list(paged.gather_kv8(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["n"]))
    return sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "plan":
        # lengths in and out, the offsets, the slot map's three arrays and the touched blocks (room for them is written whole)
        cap = min(case["room"], case["room"] // case["page"] + 2 * case["rows"])
        return {"bytes": case["rows"] * 16 + case["room"] * 16 + cap * 16, "flops": 0}
    if op == "append":
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["tokens"] * D * ((H + 2 * Hkv) * size + H * 2 + 2 * Hkv), "flops": case["tokens"] * D * (H + Hkv) * 3}
    if op == "attn":
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        lens = _lengths(case, 1)
        qn = [case["q"] if i % 3 == 0 else 1 + i % case["q"] for i in range(case["rows"])]
        return {"bytes": sum(lens) * Hkv * D * 2 + sum(qn) * H * (D * 4 + 4), "flops": sum(4 * n * q * H * D for n, q in zip(lens, qn))}
    if op == "gather":
        return {"bytes": case["longest"] * case["kv_heads"] * case["dim"] * 6, "flops": 0}
    return {"bytes": case["rows"] * case["vocab"] * (4 if case["dtype"] == "float32" else 2), "flops": 0}


# --------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rows(s, x, table_row, n):
    P = s["case"]["page"]
    blocks = -(-n // P)
    page = table_row[:blocks].long()
    rows = _take(s[x], page).double() * s[x + "_scale"][page].double()[:, :, None, None]
    return rows.permute(0, 2, 1, 3).reshape(blocks * P, rows.shape[1], rows.shape[3])[:n]


def exact(case, seed):
    if case["op"] in ("plan", "sample"):
        return None
    s = prepare(case, seed)
    if case["op"] == "gather":
        return [_exact_rows(s, x, s["table"], s["n"]).transpose(0, 1) for x in "kv"]
    if case["op"] == "append":
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        x = s["qkv"].double().view(s["tokens"], H + 2 * Hkv, D)
        c = s["cos"].double()[s["pos"].long()].repeat(1, 2).unsqueeze(1)
        d = s["sin"].double()[s["pos"].long()].repeat(1, 2).unsqueeze(1)
        q = x[:, :H]
        turned = torch.cat([-q[..., D // 2:], q[..., :D // 2]], -1)
        return {"q": q * c + turned * d, "k": None, "v": None, "k_scale": None, "v_scale": None}
    lens, cu = s["kv_len"].tolist(), s["cu"].tolist()
    H, Hkv = case["heads"], case["kv_heads"]
    os, ls = [], []
    for r in range(case["rows"]):
        q = s["q"][cu[r]:cu[r + 1]].double()
        m, n = q.shape[0], lens[r]
        if n == 0:
            os.append(torch.zeros_like(q))
            ls.append(q.new_full((H, m), float("-inf")))
            continue
        k = _exact_rows(s, "k", s["table"][r], n)
        v = _exact_rows(s, "v", s["table"][r], n)
        a = torch.einsum("ihgd,jhd->hgij", q.view(m, Hkv, H // Hkv, -1), k) * s["scale"]
        hidden = torch.arange(n, device=q.device)[None] > (n - m + torch.arange(m, device=q.device))[:, None]
        a = a.masked_fill(hidden, float("-inf"))
        lse = torch.logsumexp(a, -1)
        p = torch.exp(a - lse.unsqueeze(-1)).nan_to_num(0.0)
        os.append(torch.einsum("hgij,jhd->ihgd", p, v).reshape(m, H, -1))
        ls.append(lse.reshape(H, m))
    return {"o": torch.cat(os), "lse": torch.cat(ls, 1)}
