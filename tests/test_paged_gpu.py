"""The paged 8-bit KV cache kernels and the batched sampler on the GPU.

Integer results (plans, codes, scales, tokens) must equal the CPU oracle's bit for bit. Attention is
compared with the float64 oracle on the same cache; see `check_attention` for the tolerances.
"""

import math
import random

import pytest
import torch

from hetero_cp_ringattn_b200.config import preset
from hetero_cp_ringattn_b200.kv.quant import CODES, Kv8Cache
from hetero_cp_ringattn_b200.ops import paged, paged_reference as pref, reference as ref, sampling

pytestmark = pytest.mark.gpu


def same(a, b):
    """Bit equality of a GPU tensor and a CPU one (NaN codes included)."""
    a = a.cpu()
    if a.dtype == torch.float8_e4m3fn:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
    return torch.equal(a, b)


def status_tensor(dev):
    return torch.zeros(8, dtype=torch.int32, device=dev)


# --------------------------------------------------------------------------- step plan
def _plan_state(rows, width, page, longest, seed):
    r = random.Random(seed)
    lens = [r.choice([0, 1, page, longest, r.randrange(0, longest + 1)]) for _ in range(rows)]
    held = [-(-n // page) for n in lens]
    pages = rows * width
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    head = r.randrange(0, 5 * pages)
    ring = torch.full((pages,), -1, dtype=torch.int32)
    ring[(torch.arange(pages - at) + head) % pages] = order[at:]
    return torch.tensor(lens, dtype=torch.int32), table, ring, torch.tensor([head, head + pages - at])


@pytest.mark.parametrize("rows,width,page,room,kind", [
    (1, 4, 16, 1, "one"), (3, 8, 64, 3, "one"), (64, 9, 32, 64, "one"), (257, 5, 16, 1000, "mixed"), (4096, 3, 16, 5000, "mixed"),
    (7, 40, 16, 3001, "prompt"), (33, 300, 128, 40000, "prompt"), (5, 12, 10, 77, "mixed"), (40, 6, 16, 200, "release"),
    (9, 4, 16, 8, "toomany"), (9, 2, 16, 4000, "wide"), (6, 3, 16, 500, "nopages"), (2, 5, 64, 10, "nothing")])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_equals_the_oracle(dev, rows, width, page, room, kind, in_place):
    r = random.Random(rows + room)
    kv_len, table, ring, counters = _plan_state(rows, width, page, max(1, (width - 1) * page // 2), rows)
    free = {"one": lambda i: 1, "mixed": lambda i: r.choice([-1, 0, 1, 1, 2]), "release": lambda i: r.choice([-1, -1, 3]),
            "prompt": lambda i: r.randrange(0, max(1, min(room // rows, width * page // 2))), "toomany": lambda i: 1,
            "wide": lambda i: width * page if i == 4 else 1, "nopages": lambda i: page + 1, "nothing": lambda i: 0}[kind]
    add = torch.tensor([free(i) for i in range(rows)], dtype=torch.int32)
    if kind == "nopages":
        counters[0] = counters[1] - 2
    gpu = [x.to(dev) for x in (add, kv_len, table, ring, counters)]
    want = paged.plan_step(add, kv_len, table, ring, counters, page=page, max_tokens=room)
    out = paged.StepPlan.empty(rows, page, room, dev, kv_len=gpu[1] if in_place else None, counters=gpu[4] if in_place else None)
    got = paged.plan_step(*gpu, page=page, max_tokens=room, out=out)
    for name in ("cu", "row", "pos", "slot", "unit", "kv_len", "counters", "info"):
        assert same(getattr(got, name), getattr(want, name)), name
    assert same(gpu[2], table) and same(gpu[3], ring)
    assert int(got.info[3]) == {"toomany": 3, "wide": 2, "nopages": 1}.get(kind, 0)


@pytest.mark.parametrize("free", [0, 1, 2, 4, 9])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_gives_back_no_more_pages_than_the_ring_holds(dev, free, in_place):
    from test_paged_cpu import _crowded_ring
    add = torch.tensor([-1, 3], dtype=torch.int32)
    host = _crowded_ring(free)
    gpu = [t.to(dev) for t in host]
    # the ring lies inside a longer tensor: what stands behind it must stay
    wide = torch.full((64,), -7, dtype=torch.int32, device=dev)
    wide[:4] = gpu[2]
    gpu[2] = wide[:4]
    want = paged.plan_step(add, *host, page=16, max_tokens=8)
    out = paged.StepPlan.empty(2, 16, 8, dev, kv_len=gpu[0] if in_place else None, counters=gpu[3] if in_place else None)
    got = paged.plan_step(add.to(dev), *gpu, page=16, max_tokens=8, out=out)
    for name in ("cu", "row", "pos", "slot", "unit", "kv_len", "counters", "info"):
        assert same(getattr(got, name), getattr(want, name)), name
    assert same(gpu[1], host[1]) and same(gpu[2], host[2]) and (wide[4:] == -7).all()


def test_plan_refusals(dev):
    kv_len, table, ring, counters = (x.to(dev) for x in _plan_state(4, 3, 16, 20, 0))
    add = torch.ones(4, dtype=torch.int32, device=dev)
    good = dict(page=16, max_tokens=4)
    for bad in ((add.long(), kv_len, table, ring, counters), (add[:3], kv_len, table, ring, counters),
                (add, kv_len, table[:, ::2], ring, counters), (add, kv_len, table, ring, counters.int()),
                (add, kv_len.cpu(), table, ring, counters)):
        with pytest.raises(RuntimeError):
            paged.plan_step(*bad, **good)
    with pytest.raises(RuntimeError):
        paged.plan_step(add, kv_len, table, ring, counters, page=0, max_tokens=4, out=paged.StepPlan.empty(4, 16, 4, dev))
    with pytest.raises(RuntimeError):   # room for fewer units than the tokens can touch
        out = paged.StepPlan.empty(4, 16, 4, dev)
        out.unit = out.unit[:2].contiguous()
        paged.plan_step(add, kv_len, table, ring, counters, out=out, **good)


# --------------------------------------------------------------------------- append
def _strided_cache(pages, heads, page, dim, code, dev, spread=False):
    """A cache; `spread`: k and v interleaved in one allocation, rows further apart than their length."""
    g = torch.Generator().manual_seed(7)
    if spread:
        raw = torch.randint(0, 100, (pages, 2, heads, page, dim + 32), generator=g, dtype=torch.uint8).to(dev)
        sc = torch.ones(pages, 2, heads, device=dev) * 0.125
        k, v = (raw[:, i, :, :, :dim].view(CODES[code]) for i in (0, 1))
        return k, v, sc[:, 0], sc[:, 1]
    raw = torch.randint(0, 100, (2, pages, heads, page, dim), generator=g, dtype=torch.uint8).to(dev).view(CODES[code])
    sc = torch.ones(2, pages, heads, device=dev) * 0.125
    return raw[0], raw[1], sc[0], sc[1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code,page,heads,hkv,dim,news", [
    ("e4m3", 64, 4, 2, 128, [1, 1, 1]), ("int8", 16, 6, 2, 64, [1, 0, 1]), ("e4m3", 16, 7, 1, 128, [40, 1, 0, 17]),
    ("int8", 128, 3, 3, 128, [300, 129]), ("e4m3", 32, 16, 1, 64, [33, 5, 64]), ("int8", 64, 5, 5, 64, [2, 130, 1]),
    ("e4m3", 128, 9, 3, 64, [128, 127, 1])])
@pytest.mark.parametrize("spread", [False, True])
def test_append_equals_the_oracle(dev, dtype, code, page, heads, hkv, dim, news, spread):
    """Codes, scales and q bit for bit, over fresh and open blocks (whose stored codes are rescaled where
    the scale grows), short and long units, strided inputs and caches."""
    torch.manual_seed(sum(news) + dim)
    rows = len(news)
    old = [0, page - 1, page, page + 3][:rows]
    table = torch.randperm(rows * 8)[: rows * 8].view(rows, 8).to(torch.int32)
    pages = rows * 8
    kv_len = torch.tensor(old, dtype=torch.int32)
    plan = paged.plan_step(torch.tensor(news, dtype=torch.int32), kv_len, table.clone(), torch.arange(pages, dtype=torch.int32),
                           torch.tensor([0, pages]), page=page, max_tokens=sum(news))
    # the plan's table is not used: pages fixed beforehand
    T, width = sum(news), (heads + 2 * hkv) * dim
    buf = torch.randn(T, width + (16 if spread else 0)) * 2.0 ** torch.randint(-6, 7, (T, 1))
    buf[0] = 0.0
    x = buf[:, :width].to(dtype) if not spread else buf.to(dtype)[:, :width]
    cos, sin = ref.rope_cos_sin(torch.arange(8 * page), dim, 500000.0)
    k, v, ks, vs = _strided_cache(pages, hkv, page, dim, code, dev, spread)
    kc, vc, ksc, vsc = (t.cpu().clone() for t in (k, v, ks, vs))
    want = paged.rope_append_kv8(x, cos, sin, plan.pos, plan.unit, table, kc, vc, ksc, vsc, heads=heads)
    st = status_tensor(dev)
    xg = buf.to(dtype).to(dev)[:, :width] if spread else x.to(dev)
    got = paged.rope_append_kv8(xg, cos.to(dev), sin.to(dev), plan.pos.to(dev), plan.unit.to(dev), table.to(dev), k, v, ks, vs,
                                heads=heads, status=st)
    assert same(got, want)
    for a, b in ((ks, ksc), (vs, vsc), (k, kc), (v, vc)):
        assert same(a.contiguous() if a.dtype == torch.float32 else a, b)
    assert int(st[0]) == 0


def test_append_non_finite_inputs(dev):
    """NaN keeps its place in e4m3 and becomes 0 in int8, infinities saturate at the largest scale, and
    neither touches another head's or block's codes."""
    for code in ("e4m3", "int8"):
        k, v, ks, vs = _strided_cache(4, 2, 16, 64, code, dev)
        kc, vc, ksc, vsc = (t.cpu().clone() for t in (k, v, ks, vs))
        x = torch.randn(5, (2 + 4) * 64)
        x[1, 2 * 64 + 5] = float("nan")
        x[2, 4 * 64 + 7] = float("inf")
        unit = torch.tensor([[0, 0, 5, 2]], dtype=torch.int32)
        pos = torch.arange(2, 7, dtype=torch.int32)
        table = torch.tensor([[3]], dtype=torch.int32)
        cos, sin = ref.rope_cos_sin(torch.arange(16), 64, 10000.0)
        paged.rope_append_kv8(x, cos, sin, pos, unit, table, kc, vc, ksc, vsc, heads=2)
        paged.rope_append_kv8(x.to(dev), cos.to(dev), sin.to(dev), pos.to(dev), unit.to(dev), table.to(dev), k, v, ks, vs, heads=2)
        assert same(ks, ksc) and same(vs, vsc) and same(v, vc)
        got, want = k.cpu().float(), kc.float()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_append_reports_and_skips_bad_places(dev):
    k, v, ks, vs = _strided_cache(2, 1, 16, 64, "e4m3", dev)
    before = k.clone().view(torch.uint8)
    x = torch.randn(2, 3 * 64, device=dev)
    cos, sin = (t.to(dev) for t in ref.rope_cos_sin(torch.arange(16), 64, 10000.0))
    for unit, table, pos in (([[0, 0, 2, 0]], [[7]], [0, 1]), ([[0, 0, 2, 0]], [[-1]], [0, 1]), ([[3, 0, 2, 0]], [[1]], [0, 1]),
                             ([[0, 0, 2, 15]], [[1]], [0, 1]), ([[0, 1, 2, 0]], [[1]], [0, 1]), ([[0, 0, 2, 16]], [[1]], [0, 1])):
        st = status_tensor(dev)
        paged.rope_append_kv8(x, cos, sin, torch.tensor(pos, dtype=torch.int32, device=dev),
                              torch.tensor(unit, dtype=torch.int32, device=dev), torch.tensor(table, dtype=torch.int32, device=dev),
                              k, v, ks, vs, heads=1, status=st)
        assert int(st[0]) == 18 and torch.equal(k.view(torch.uint8), before)


@pytest.mark.parametrize("dtype,code,page,heads,hkv,dim,old,news", [
    # many blocks: teams that go through several KV heads, the next one's values fetched ahead
    (torch.bfloat16, "e4m3", 64, 8, 8, 128, [0, 37, 63, 1], [9000, 5001, 1500, 900]),
    (torch.bfloat16, "int8", 64, 4, 5, 128, [17, 0], [9000, 3333]),          # 5 heads: a last group of fewer
    (torch.float32, "e4m3", 64, 3, 3, 64, [5], [20011]),
    (torch.float16, "int8", 128, 2, 7, 64, [127, 3], [20000, 801]),
    # several teams a CTA (pages of 16 and 32), whole blocks and open ones, one head and several
    (torch.bfloat16, "e4m3", 16, 4, 2, 128, [0, 15], [160, 97]), (torch.float32, "int8", 16, 2, 3, 64, [9], [333]),
    (torch.float16, "e4m3", 32, 4, 1, 128, [31, 2, 0], [64, 500, 33]), (torch.bfloat16, "int8", 32, 2, 6, 64, [1], [1000]),
    (torch.bfloat16, "e4m3", 16, 2, 8, 64, [3, 0], [9001, 4000]), (torch.float32, "e4m3", 32, 2, 5, 128, [30], [9999]),
    (torch.float32, "int8", 16, 2, 7, 128, [8], [7000])])
def test_append_of_prompts_equals_the_oracle(dev, dtype, code, page, heads, hkv, dim, old, news):
    """Prompts of whole blocks behind open ones, whose stored codes are rescaled: codes, scales and q bit
    for bit, with nothing else in the cache changed."""
    g = torch.Generator().manual_seed(page + hkv + dim)
    rows, width = len(old), max(-(-(o + n) // page) for o, n in zip(old, news)) + 1
    pages = rows * width + 3
    table = torch.randperm(pages, generator=g)[:rows * width].view(rows, width).to(torch.int32)
    units, pos, t = [], [], 0
    for r, (o, n) in enumerate(zip(old, news)):
        p = o
        while p < o + n:
            m = min(o + n, (p // page + 1) * page) - p
            units.append([r, t, m, p])
            t, p = t + m, p + m
        pos.append(torch.arange(o, o + n))
    T, unit, pos = t, torch.tensor(units, dtype=torch.int32), torch.cat(pos).to(torch.int32)
    assert T >= 12 * len(units)
    x = (torch.randn(T, (heads + 2 * hkv) * dim, generator=g) * 2.0 ** torch.randint(-4, 5, (T, 1), generator=g)).to(dtype)
    cos, sin = ref.rope_cos_sin(torch.arange(width * page), dim, 500000.0)
    k, v, ks, vs = _strided_cache(pages, hkv, page, dim, code, dev)
    kc, vc, ksc, vsc = (c.cpu().clone() for c in (k, v, ks, vs))
    want = paged.rope_append_kv8(x, cos, sin, pos, unit, table, kc, vc, ksc, vsc, heads=heads)
    st = status_tensor(dev)
    got = paged.rope_append_kv8(x.to(dev), cos.to(dev), sin.to(dev), pos.to(dev), unit.to(dev), table.to(dev), k, v, ks, vs,
                                heads=heads, status=st)
    assert same(got, want) and int(st[0]) == 0
    for a, b in ((ks, ksc), (vs, vsc), (k, kc), (v, vc)):
        assert same(a, b)


@pytest.mark.parametrize("n,page", [(2, 16), (16, 16), (33, 64)])
@pytest.mark.parametrize("shift", [-1, 1])
def test_append_writes_nothing_past_the_rotary_tables(dev, n, page, shift):
    """Row 0's positions leave the tables (at their end by one, or below 0), row 1's are good: row 0's codes,
    scales and neighbours stay, its q is 0 where the position is bad, and row 1 is as alone. Units of 2
    tokens take the short form, those of 16 and more the block form."""
    tab = page // 2 + n
    p0 = page // 2 + 1 if shift > 0 else -1
    if shift > 0 and p0 % page + n > page:
        p0, tab = page, page + n - 1                    # a whole block that ends one past the tables
    k, v, ks, vs = _strided_cache(4, 2, page, 64, "e4m3", dev)
    cos, sin = (t.to(dev) for t in ref.rope_cos_sin(torch.arange(tab), 64, 10000.0))
    x = torch.randn(2 * n, (2 + 4) * 64, device=dev)
    pos = torch.cat([torch.arange(p0, p0 + n), torch.arange(n)]).to(torch.int32).to(dev)
    unit = torch.tensor([[0, 0, n, p0], [1, n, n, 0]], dtype=torch.int32, device=dev)
    table = torch.tensor([[3, 1], [2, 0]], dtype=torch.int32, device=dev)
    want = [t.clone() for t in (k, v, ks, vs)]
    want_q = paged.rope_append_kv8(x[n:], cos, sin, pos[n:], unit[1:] - torch.tensor([0, n, 0, 0], device=dev, dtype=torch.int32),
                                   table, *want, heads=2)
    st = status_tensor(dev)
    q = paged.rope_append_kv8(x, cos, sin, pos, unit, table, k, v, ks, vs, heads=2, status=st)
    assert int(st[0]) == 18
    for a, b in zip((k, v, ks, vs), want):
        assert same(a, b.cpu())
    bad = (pos < 0) | (pos >= tab)
    assert bad.any() and (q[bad] == 0).all() and (q[:n][~bad[:n]] != 0).any() and torch.equal(q[n:], want_q)


def test_append_refusals(dev):
    k, v, ks, vs = _strided_cache(2, 1, 16, 64, "e4m3", dev)
    cos, sin = (t.to(dev) for t in ref.rope_cos_sin(torch.arange(16), 64, 10000.0))
    x = torch.randn(2, 3 * 64, device=dev)
    pos = torch.arange(2, dtype=torch.int32, device=dev)
    unit, table = torch.tensor([[0, 0, 2, 0]], dtype=torch.int32, device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev)
    for args, kw in (((x, cos, sin, pos, unit, table, k, v, ks, vs), dict(heads=2)),
                     ((x.double(), cos, sin, pos, unit, table, k, v, ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos[:1], unit, table, k, v, ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos, unit[:, :3].contiguous(), table, k, v, ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos, unit, table, k, v.view(torch.int8), ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos, unit, table, k.view(torch.uint8), v.view(torch.uint8), ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos, unit, table, k[:, :, :12], v[:, :, :12], ks, vs), dict(heads=1)),
                     ((x, cos, sin, pos, unit, table, k, v, ks.double(), vs.double()), dict(heads=1)),
                     ((x[:, ::1], cos[:, ::2], sin[:, ::2], pos, unit, table, k, v, ks, vs), dict(heads=1))):
        with pytest.raises(RuntimeError):
            paged.rope_append_kv8(*args, **kw)


# --------------------------------------------------------------------------- attention
def _cache(lens, page, hkv, dim, code, dev, seed=0, garbage=True):
    """Pages in random order with values of unit spread. `garbage`: every place behind a row's end, and
    every page of no row, holds NaN codes (e4m3) or the largest ones (int8)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(held + [1])), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    amp, s0 = (60.0, -6) if code == "e4m3" else (30.0, -5)
    out = []
    for _ in "kv":
        x = torch.randn(pages, hkv, page, dim, generator=g, device=dev) * amp
        data = pref.encode(x, CODES[code])
        if garbage:
            raw = data.view(torch.uint8)
            keep = torch.zeros(pages, page, dtype=torch.bool)
            for i, n in enumerate(lens):
                for b in range(held[i]):
                    keep[table[i, b], : max(0, min(page, n - b * page))] = True
            raw[~keep.to(dev).unsqueeze(1).expand(pages, hkv, page)] = 0x7F
        out.append(data)
    scales = [2.0 ** torch.randint(s0 - 2, s0 + 3, (pages, hkv), generator=g, device=dev).float() for _ in "kv"]
    return out[0], out[1], scales[0], scales[1], table.to(dev)


def check_attention(q, k, v, ks, vs, table, lens, cu, scale=None, **kw):
    """o and lse against float64. The outputs' rounding is at most 2^-8 (bf16: 8 significant bits, half a
    unit of the last at the low end of a binade) or 2^-11 (f16: 11 bits) of the value; P's
    rounding to f16 moves o by at most 2^-11 of A = sum p |v|, and float32 accumulation and the
    approximate exponential stay below that; a score sums D products in float32 and is off by at
    most about 2^-20 of sum |q k| scale, which is also lse's error."""
    dev = q.device
    scale = scale or 1.0 / math.sqrt(q.shape[-1])
    kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    most = 1 if cu is None else max(b - a for a, b in zip(cu, cu[1:]))
    st = status_tensor(dev)
    o, lse = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cut, max_q=max(1, most), scale=scale, status=st, **kw)
    assert int(st[0]) == 0, st.tolist()
    want_o, want_l = pref.attention_kv8(q, k, v, ks, vs, table, kv_len, cut, scale, dtype=torch.float64)
    mag_o, _ = pref.attention_kv8(q, k, _abs(v), ks, vs, table, kv_len, cut, scale, dtype=torch.float64)
    room = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    assert torch.equal(torch.isinf(lse), torch.isinf(want_l))
    fin = torch.isfinite(want_l)
    big = _score_size(q, k, ks, table, lens, cu, scale)
    assert ((lse.double() - want_l).abs()[fin] <= 2.0 ** -19 * (1 + big.t()[fin])).all()
    err = (o.double() - want_o).abs()
    bound = want_o.abs() * room * 1.01 + mag_o * (2.0 ** -10 + 2.0 ** -19 * big.unsqueeze(-1)) + 1e-30
    assert (err <= bound).all(), float((err / bound).max())
    assert (o.transpose(0, 1)[~fin] == 0).all()
    return o, lse


def _abs(v):
    return (v.view(torch.uint8) & 0x7F).view(v.dtype) if v.dtype == torch.float8_e4m3fn else v.abs()


def _score_size(q, k, ks, table, lens, cu, scale):
    """Largest sum |q k| scale of every (token, head)."""
    out = torch.zeros(q.shape[0], q.shape[1], dtype=torch.float64, device=q.device)
    bounds = cu or list(range(len(lens) + 1))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        kk = pref.cached_rows(_abs(k), ks, table[b], n, torch.float64).repeat_interleave(q.shape[1] // k.shape[1], dim=1)
        for t in range(bounds[b], bounds[b + 1]):
            out[t] = torch.einsum("hd,nhd->hn", q[t].double().abs(), kk).amax(1) * scale
    return out


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,hkv,dim,page", [(8, 2, 128, 64), (8, 8, 64, 16), (14, 2, 64, 32), (7, 1, 128, 128), (16, 1, 128, 16),
                                                (20, 1, 64, 64), (48, 1, 128, 32), (12, 4, 64, 128)])
def test_attention_single_tokens(dev, code, heads, hkv, dim, page):
    """GQA groups of 1 to 48, lengths of 0, 1 and around pages and tiles, garbage behind every end."""
    lens = [0, 1, 2, page - 1, page, page + 1, 31, 32, 33, 63, 65, 200, 517, 0, 1000]
    torch.manual_seed(heads + dim)
    q = (torch.randn(len(lens), heads, dim, device=dev) * 1.5).bfloat16()
    check_attention(q, *_cache(lens, page, hkv, dim, code, dev, seed=page), lens, None)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,hkv,dim,page,most", [(8, 2, 128, 64, 3), (28, 4, 128, 32, 5), (16, 2, 64, 16, 5), (4, 4, 64, 64, 9),
                                                     (32, 8, 128, 16, 4), (8, 1, 64, 128, 16), (2, 2, 128, 16, 70)])
def test_attention_ragged_query_tokens(dev, code, heads, hkv, dim, page, most):
    """1 to 70 query tokens a request, causal among themselves, more of them than cached rows, none at
    all, and tokens that see nothing."""
    r = random.Random(heads + most)
    lens = [0, 1, most, most - 1, 33, 64, 65, 300, 129, 513, 2, 96]
    qn = [1, most, most, most, 0, 1, most, r.randrange(1, most + 1), most, 2, most, 3]
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    torch.manual_seed(most)
    q = (torch.randn(cu[-1], heads, dim, device=dev) * 1.5).bfloat16()
    check_attention(q, *_cache(lens, page, hkv, dim, code, dev, seed=most), lens, cu)


@pytest.mark.parametrize("max_q", [1, 2, 3])
@pytest.mark.parametrize("heads,hkv,dim", [(8, 2, 128), (4, 4, 64)])
def test_attention_results_do_not_depend_on_max_q(dev, heads, hkv, dim, max_q):
    """Requests with more query tokens than max_q says (it defaults to 1): the causal limits, and every
    query row of a request that many CTAs share."""
    lens, qn = [9, 3000, 40, 6, 2500], [5, 5, 0, 9, 33]
    cu = [0]
    for n in qn:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], heads, dim, device=dev).bfloat16()
    k, v, ks, vs, table = _cache(lens, 32, hkv, dim, "e4m3", dev)
    kv_len, cut = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, cu))
    want, want_l = check_attention(q, k, v, ks, vs, table, lens, cu)
    st = status_tensor(dev)
    kw = {} if max_q == 1 else dict(max_q=max_q)
    got, got_l = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cut, status=st, **kw)
    assert int(st[0]) == 0
    assert torch.equal(torch.isinf(got_l), torch.isinf(want_l))
    # each call's o is within one rounding of the exact value and 2^-10 of sum p |v| (at most max |v|)
    top = float((_abs(v).float().nan_to_num(0.0).clamp(max=400.0) * vs.view(*vs.shape, 1, 1)).max())
    assert ((got.float() - want.float()).abs() <= 2 * (2.0 ** -8 * want.float().abs() + 2.0 ** -10 * top)).all()
    assert ((got_l - want_l)[torch.isfinite(want_l)].abs() <= 1e-4).all()


def test_attention_query_offsets_past_the_tokens_are_reported(dev):
    lens = [40, 50]
    k, v, ks, vs, table = _cache(lens, 16, 1, 64, "e4m3", dev)
    q = torch.randn(3, 2, 64, device=dev).bfloat16()
    for cu, bad in (([0, 2, 3], False), ([0, 2, 5], True), ([-1, 2, 3], True), ([0, 2, 1], True)):
        st = status_tensor(dev)
        o, _ = paged.attention_kv8(q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device=dev),
                                   torch.tensor(cu, dtype=torch.int32, device=dev), max_q=3, status=st)
        assert (int(st[0]) == 18) == bad and torch.isfinite(o).all()


@pytest.mark.parametrize("batch,longest", [(1, 20011), (3, 9000), (40, 700), (300, 90), (1024, 40)])
def test_attention_work_split(dev, batch, longest):
    """One long request (every CTA on the same heads) to more requests than CTAs."""
    r = random.Random(batch)
    lens = [longest] + [r.randrange(0, longest + 1) for _ in range(batch - 1)]
    q = torch.randn(batch, 8, 64, device=dev).bfloat16()
    check_attention(q, *_cache(lens, 32, 2, 64, "e4m3", dev), lens, None)


def test_attention_types_strides_and_scales(dev):
    """f16 q, q as a slice of wider rows, a strided cache, scales of any positive size (far apart within a
    row), and a query row of zeros."""
    lens, page, hkv, dim = [100, 333, 65], 32, 2, 128
    k, v, ks, vs, table = _cache(lens, page, hkv, dim, "e4m3", dev)
    wide = torch.randn(3, 8 * dim + 40, device=dev).half()
    q = wide[:, 8:8 + 8 * dim].view(3, 8, dim)
    q[1, 3] = 0
    check_attention(q, k, v, ks, vs, table, lens, None)
    room = torch.zeros(k.shape[0], 2, hkv, page, dim + 16, dtype=torch.uint8, device=dev)
    ks2 = torch.zeros(k.shape[0], 2, hkv, device=dev)
    for i, (src, sc) in enumerate(((k, ks), (v, vs))):
        room[:, i, :, :, :dim] = src.view(torch.uint8)
        ks2[:, i] = sc * 1.37
    kk, vv = (room[:, i, :, :, :dim].view(torch.float8_e4m3fn) for i in (0, 1))
    check_attention(q, kk, vv, ks2[:, 0], ks2[:, 1], table, lens, None)
    g = torch.Generator(device=dev).manual_seed(3)
    far = 2.0 ** torch.randint(-30, 30, vs.shape, generator=g, device=dev).float()
    check_attention(q.bfloat16(), k, v, ks, far, table, lens, None)     # (values past f16's range)


def test_attention_zero_scale_block(dev):
    """A block of V scaled by 0 adds its weight and no value; a K block scaled by 0 gives scores of 0."""
    lens = [130]
    k, v, ks, vs, table = _cache(lens, 32, 1, 64, "e4m3", dev)
    vs[table[0, 1]] = 0.0
    ks[table[0, 2]] = 0.0
    check_attention(torch.randn(1, 4, 64, device=dev).bfloat16(), k, v, ks, vs, table, lens, None)


@pytest.mark.parametrize("heads,most", [(2, 3), (8, 5)])
def test_attention_nan_of_a_later_token_stays_out_of_earlier_ones(dev, heads, most):
    """The last query token's own K and V are NaN: only that token's output is."""
    n = 70
    k, v, ks, vs, table = _cache([n], 32, 2, 64, "e4m3", dev)
    q = torch.randn(most, heads, 64, device=dev).bfloat16()
    kv_len, cu = torch.tensor([n], dtype=torch.int32, device=dev), torch.tensor([0, most], dtype=torch.int32, device=dev)
    clean, _ = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cu, max_q=most)
    for t in (k, v):
        t.view(torch.uint8)[table[0, (n - 1) // 32], :, (n - 1) % 32] = 0x7F
    o, lse = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cu, max_q=most)
    assert torch.equal(o[:-1], clean[:-1]) and torch.isfinite(lse[:, :-1]).all()
    assert torch.isnan(o[-1]).all() and torch.isnan(lse[:, -1]).all()


def test_attention_non_finite_query_row(dev):
    """An infinite and a NaN query element make their own (token, head) NaN and no other."""
    lens = [90, 40]
    k, v, ks, vs, table = _cache(lens, 16, 1, 128, "int8", dev)
    q = torch.randn(2, 8, 128, device=dev).bfloat16()
    kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    clean, _ = paged.attention_kv8(q, k, v, ks, vs, table, kv_len)
    q[0, 2, 5], q[1, 7, 0] = float("inf"), float("nan")
    o, _ = paged.attention_kv8(q, k, v, ks, vs, table, kv_len)
    bad = torch.zeros(2, 8, dtype=torch.bool, device=dev)
    bad[0, 2] = bad[1, 7] = True
    assert torch.isnan(o[bad]).all() and torch.isfinite(o[~bad]).all()
    assert ((o[~bad].float() - clean[~bad].float()).abs() <= 2.0 ** -7 * clean[~bad].float().abs() + 1e-3).all()


def test_attention_page_ids_out_of_range_are_reported(dev):
    k, v, ks, vs, table = _cache([100], 16, 1, 64, "e4m3", dev, garbage=False)
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 3] = bad
        st = status_tensor(dev)
        o, _ = paged.attention_kv8(torch.randn(1, 2, 64, device=dev).bfloat16(), k, v, ks, vs, t,
                                   torch.tensor([100], dtype=torch.int32, device=dev), status=st)
        assert int(st[0]) == 18 and int(st[2]) == bad and torch.isfinite(o).all()


def test_attention_of_other_requests_does_not_depend_on_a_report(dev):
    """A status word that is set already, and a bad page id of one request, leave the others' outputs as
    they are (and the first report stands)."""
    lens = [3000, 20000, 700, 5000]
    k, v, ks, vs, table = _cache(lens, 16, 2, 128, "e4m3", dev, garbage=False)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    for heads, most in ((8, 1), (16, 3)):
        cu = torch.arange(0, 4 * most + 1, most, dtype=torch.int32, device=dev)
        q = torch.randn(4 * most, heads, 128, device=dev).bfloat16()
        want, want_l = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cu, max_q=most)
        st = status_tensor(dev)
        st[0] = 99
        got, got_l = paged.attention_kv8(q, k, v, ks, vs, table, kv_len, cu, max_q=most, status=st)
        assert torch.equal(got, want) and torch.equal(got_l, want_l) and st.tolist() == [99] + [0] * 7
        bad = table.clone()
        bad[1, ::7] = -1
        st = status_tensor(dev)
        got, got_l = paged.attention_kv8(q, k, v, ks, vs, bad, kv_len, cu, max_q=most, status=st)
        assert int(st[0]) == 18 and int(st[1]) == 411
        rows = [t for t in range(4 * most) if t // most != 1]
        assert torch.equal(got[rows], want[rows]) and torch.equal(got_l[:, rows], want_l[:, rows])


def test_attention_lengths_past_the_table_are_cut(dev):
    k, v, ks, vs, table = _cache([64], 16, 1, 64, "e4m3", dev)
    q = torch.randn(1, 2, 64, device=dev).bfloat16()
    a, _ = paged.attention_kv8(q, k, v, ks, vs, table, torch.tensor([64], dtype=torch.int32, device=dev))
    b, _ = paged.attention_kv8(q, k, v, ks, vs, table, torch.tensor([1 << 30], dtype=torch.int32, device=dev))
    c, l = paged.attention_kv8(q, k, v, ks, vs, table, torch.tensor([-5], dtype=torch.int32, device=dev))
    assert torch.equal(a, b) and (c == 0).all() and torch.isinf(l).all()


def test_attention_past_32_bit_offsets(dev):
    """Pages behind the first 4 GiB of each of K and V."""
    hkv, page, dim = 8, 128, 128
    pages = (1 << 32) // (hkv * page * dim) + 40
    k = torch.empty(pages, hkv, page, dim, dtype=torch.int8, device=dev)
    v = torch.empty_like(k)
    ks = torch.full((pages, hkv), 2.0 ** -5, device=dev)
    vs = ks * 2
    ids = [pages - 1, 3, pages - 17, pages - 2]
    for i in ids:
        k[i] = torch.randint(-90, 90, k[i].shape, device=dev, dtype=torch.int8)
        v[i] = torch.randint(-90, 90, k[i].shape, device=dev, dtype=torch.int8)
    table = torch.tensor([ids], dtype=torch.int32, device=dev)
    q = torch.randn(1, 16, dim, device=dev).bfloat16()
    check_attention(q, k, v, ks, vs, table, [500], None)
    kb, vb = paged.gather_kv8(k, v, ks, vs, table[0], 500)
    assert torch.equal(kb, pref.cached_rows(k, ks, table[0], 500).transpose(0, 1).bfloat16())
    assert torch.equal(vb, pref.cached_rows(v, vs, table[0], 500).transpose(0, 1).bfloat16())


def test_attention_shards_merge(dev):
    """The two halves of a request's pages attended separately and merged by their lse equal the whole."""
    n, page = 640, 64
    k, v, ks, vs, table = _cache([n], page, 2, 64, "e4m3", dev)
    q = torch.randn(1, 8, 64, device=dev).half()
    whole, wl = check_attention(q, k, v, ks, vs, table, [n], None)
    parts = [paged.attention_kv8(q, k, v, ks, vs, t.contiguous(), torch.tensor([m], dtype=torch.int32, device=dev))
             for t, m in ((table[:, :4], 256), (table[:, 4:], n - 256), (table[:, :1], 0))]
    o, l = ref.merge_partials([p[0].double() for p in parts], [p[1].double() for p in parts])
    assert (l - wl.double()).abs().max() < 1e-5
    assert (o - whole.double()).abs().max() <= 3 * 2.0 ** -11 * whole.double().abs().max()


def test_attention_streams_do_not_share_workspaces(dev):
    """Calls in flight on two streams at once, each with its own requests."""
    cases = []
    for s in range(2):
        lens = [3000 + 500 * s, 17, 900]
        cases.append((torch.randn(3, 8, 128, device=dev).bfloat16(), *_cache(lens, 64, 2, 128, "int8", dev, seed=s),
                      torch.tensor(lens, dtype=torch.int32, device=dev)))
    want = [paged.attention_kv8(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged.attention_kv8(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def test_attention_and_gather_refusals(dev):
    k, v, ks, vs, table = _cache([40, 20], 16, 2, 64, "e4m3", dev)
    kv_len = torch.tensor([40, 20], dtype=torch.int32, device=dev)
    q = torch.randn(2, 4, 64, device=dev).bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    for args, kw in (((q.float(), k, v, ks, vs, table, kv_len), {}), ((q[:, :3], k, v, ks, vs, table, kv_len), {}),
                     ((q[:1], k, v, ks, vs, table, kv_len), {}), ((q, k, v, ks, vs, table, kv_len.long()), {}),
                     ((q, k, v, ks, vs, table[:1], kv_len), {}), ((q, k, v, ks, vs, table, kv_len, cu[:2]), dict(max_q=1)),
                     ((q, k, v, ks, vs, table, kv_len, cu), dict(max_q=0)), ((q, k, v, ks[:1], vs[:1], table, kv_len), {}),
                     ((q, k[:, :, :, 1:], v[:, :, :, 1:], ks, vs, table, kv_len), {}),
                     ((q, k, v, ks, vs, table, kv_len), dict(out=torch.empty(2, 4, 64, device=dev)))):
        with pytest.raises(RuntimeError):
            paged.attention_kv8(*args, **kw)
    with pytest.raises(RuntimeError):
        paged.gather_kv8(k, v, ks, vs, table[0], 16 * table.shape[1] + 1)
    with pytest.raises(RuntimeError):
        paged.gather_kv8(k, v, ks, vs, table, 4)
    with pytest.raises(RuntimeError):
        paged.gather_kv8(k, v, ks, vs, table[0], 20, out=(torch.empty(2, 19, 64, device=dev, dtype=torch.bfloat16),) * 2)
    o, _ = paged.attention_kv8(q[:0], k, v, ks, vs, table, kv_len, torch.zeros(3, dtype=torch.int32, device=dev))
    assert o.shape == (0, 4, 64)


@pytest.mark.parametrize("shape", [(2, 0, 16, 64), (0, 1, 16, 64), (2, 1, 0, 64), (2, 1, 16, 0)])
def test_empty_caches_are_refused(dev, shape):
    k, v = (torch.zeros(shape, dtype=torch.int8, device=dev) for _ in "kv")
    ks, vs = (torch.ones(shape[:2], device=dev) for _ in "kv")
    table, n = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 4, shape[3], dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="the cache must have"):
        paged.attention_kv8(q, k, v, ks, vs, table, n, scale=1.0)
    with pytest.raises(RuntimeError, match="the cache must have"):
        paged.gather_kv8(k, v, ks, vs, table[0], 1)
    tab = torch.zeros(4, shape[3] // 2, device=dev)
    with pytest.raises(RuntimeError, match="the cache must have"):
        paged.rope_append_kv8(torch.zeros(1, (4 + 2 * shape[1]) * shape[3], device=dev), tab, tab, n,
                              torch.zeros(1, 4, dtype=torch.int32, device=dev), table, k, v, ks, vs, heads=4)


def test_sizes_past_32_bit_numbers_are_refused(dev):
    """A gather of 2^28 rows of 128 dims (2^31 pieces of 16 bytes), and a plan of 2^30 tokens: refused before
    anything of that size is allocated or launched."""
    k, v = (torch.zeros(1, 1, 128, 128, dtype=torch.int8, device=dev) for _ in "kv")
    ks, vs = (torch.ones(1, 1, device=dev) for _ in "kv")
    with pytest.raises(RuntimeError, match="rows to gather out of range"):
        paged.gather_kv8(k, v, ks, vs, torch.zeros(1 << 21, dtype=torch.int32, device=dev), 1 << 28)
    i32 = dict(dtype=torch.int32, device=dev)
    T = 1 << 30
    many = torch.empty(T, **i32)
    out = paged.StepPlan(cu=torch.empty(2, **i32), row=many, pos=many, slot=torch.empty(T, dtype=torch.int64, device=dev),
                         unit=torch.empty(1026, 4, **i32), kv_len=torch.empty(1, **i32),
                         counters=torch.empty(2, dtype=torch.int64, device=dev), info=torch.empty(4, **i32))
    with pytest.raises(RuntimeError, match="fewer than 2\\^30 tokens"):
        paged.plan_step(torch.ones(1, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32),
                        torch.tensor([0, 1], device=dev), page=1 << 20, max_tokens=T, out=out)


# --------------------------------------------------------------------------- gather
@pytest.mark.parametrize("code,page,hkv,dim,n", [("e4m3", 16, 1, 64, 1), ("int8", 64, 3, 128, 200), ("e4m3", 128, 8, 64, 1000),
                                                 ("int8", 32, 2, 64, 33), ("e4m3", 64, 2, 128, 0)])
def test_gather_equals_the_oracle(dev, code, page, hkv, dim, n):
    k, v, ks, vs, table = _cache([max(n, 1)], page, hkv, dim, code, dev)
    ks *= 1.3                                   # any scale: one rounding to bf16
    out = tuple(torch.full((hkv, n + 5, dim), 7.0, dtype=torch.bfloat16, device=dev) for _ in "kv")
    kb, vb = paged.gather_kv8(k, v, ks, vs, table[0], n, out=out)
    assert torch.equal(kb[:, :n], pref.cached_rows(k, ks, table[0], n).transpose(0, 1).bfloat16() if n else kb[:, :0])
    assert torch.equal(vb[:, :n], pref.cached_rows(v, vs, table[0], n).transpose(0, 1).bfloat16() if n else vb[:, :0])
    assert (kb[:, n:] == 7).all() and (vb[:, n:] == 7).all()


# --------------------------------------------------------------------------- sampling
def _logits(kind, rows, vocab, g, dev):
    x = torch.randn(rows, vocab, generator=g, device=dev) * 2
    if kind == "flat":
        x.zero_()
    elif kind == "ties":
        x = torch.randint(0, 4, (rows, vocab), generator=g, device=dev).float()
    elif kind == "peak":
        x[:, vocab // 3] = 40
    elif kind == "masked":
        x[torch.rand(rows, vocab, generator=g, device=dev) < 0.5] = float("-inf")
    elif kind == "lowest":
        x.fill_(torch.finfo(torch.float32).min)
        x[0, vocab // 2] = float("nan")
    elif kind == "nothing":
        x.fill_(float("-inf"))
        x[-1, 0] = float("inf")
    elif kind == "tiny":
        x *= 1e-38
    return x


@pytest.mark.parametrize("kind", ["normal", "flat", "ties", "peak", "masked", "lowest", "nothing", "tiny"])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 5001, 32000, 151936])
def test_sample_equals_the_oracle(dev, kind, vocab):
    g = torch.Generator(device=dev).manual_seed(vocab)
    for rows, dtype in ((3, torch.float32), (2, torch.bfloat16)):
        x = _logits(kind, rows, vocab, g, dev).to(dtype)
        u = torch.rand(rows, generator=g, device=dev)
        for s in ((1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (2.0, 3000, 0.99, 0.01), (0.0, 5, 0.5, 0.0),
                  (1.5, max(1, vocab // 2), 0.5, 0.0), (1e-3, 0, 0.3, 0.0), (5.0, 0, 0.999, 0.2), (1e30, 0, 0.6, 0.0),
                  (float("inf"), 7, 1.0, 1.0)):
            assert same(sampling.sample(x, u, *s), sampling.sample(x.cpu(), u.cpu(), *s)), s


@pytest.mark.parametrize("kind", ["normal", "ties", "one_thread", "flat", "far", "nan"])
@pytest.mark.parametrize("vocab", [301, 513, 20481, 151936])
def test_sample_top_k_sizes(dev, kind, vocab):
    """k from 1 to past what one CTA orders: ties across the cut, the largest tokens all a fixed stride
    apart (in one thread's share), rows as good as flat, tokens with weight 0 inside the top k, NaN."""
    g = torch.Generator(device=dev).manual_seed(vocab + len(kind))
    x = torch.randn(2, vocab, generator=g, device=dev) * 3
    if kind == "ties":
        x = (x * 2).round() / 2
    elif kind == "one_thread":
        x[:, ::2048] += 30
    elif kind == "flat":
        x *= 1e-4
    elif kind == "far":
        x[:, 17:] -= 500
    elif kind == "nan":
        x[:, ::3] = float("nan")
    u = torch.rand(2, generator=g, device=dev)
    for k in (1, 2, 16, 40, 255, 256, 257, 511, 513):
        for s in ((1.0, k, 1.0, 0.0), (0.6, k, 0.9, 0.0), (3.0, k, 0.7, 0.01)):
            assert same(sampling.sample(x, u, *s), sampling.sample(x.cpu(), u.cpu(), *s)), (k, s)


def test_sample_large_vocabulary_strides_and_row_settings(dev):
    """The longest rows, rows that do not start on 16 bytes, and a row of settings each."""
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(2, 720896, generator=g, device=dev) * 2
    u = torch.rand(2, generator=g, device=dev)
    assert same(sampling.sample(x, u, 0.9, 40, 0.9), sampling.sample(x.cpu(), u.cpu(), 0.9, 40, 0.9))
    wide = torch.randn(6, 5003, generator=g, device=dev)
    x = wide[:, 1:5002]
    u = torch.tensor([0.0, 0.2, 0.5, 0.99999994, 1.0, 0.7], device=dev)
    t = torch.tensor([0.0, 0.5, 1.0, 1.3, 2.0, -1.0], device=dev)
    k = torch.tensor([3, 0, 100, 4000, 9999, -2], dtype=torch.int32, device=dev)
    p = torch.tensor([0.5, 0.9, 1.0, 0.0, 0.7, 2.0], device=dev)
    m = torch.tensor([0.0, 0.1, 0.0, -1.0, 0.5, 3.0], device=dev)
    assert same(sampling.sample(x, u, t, k, p, m), sampling.sample(x.cpu(), u.cpu(), t.cpu(), k.cpu(), p.cpu(), m.cpu()))


@pytest.mark.parametrize("u", [1.0 - 2.0 ** -24, 1.0 - 2.0 ** -23, 1.0, float("nan"), -0.5])
def test_sample_ends_of_the_uniform_range(dev, u):
    """Every row drawn at the end of its range: the last kept tokens' weights decide."""
    g = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn(300, 2000, generator=g, device=dev) * 4
    x[0, 1:], x[0, 1] = float("-inf"), x[0, 0] - 16.23
    v = torch.full((300,), u, device=dev)
    for s in ((1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0)):
        assert same(sampling.sample(x, v, *s), sampling.sample(x.cpu(), v.cpu(), *s))


def test_sample_frequencies(dev):
    """200,000 draws from one row: every token's count within 5 standard deviations of its share
    (64 tokens: a chance of 4e-5 that any is outside)."""
    n = 200000
    row = torch.randn(64, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    u = torch.rand(n, device=dev, generator=torch.Generator(device=dev).manual_seed(5))
    got = torch.bincount(sampling.sample(row.expand(n, 64), u, 0.8), minlength=64).double()
    p = torch.softmax(row.double() / 0.8, 0)
    assert ((got - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()


def test_sample_refusals(dev):
    x, u = torch.randn(2, 10, device=dev), torch.rand(2, device=dev)
    for args in ((x[0], u), (x.half(), u), (x, u[:1]), (x, u.double()), (x, u, torch.ones(3, device=dev)),
                 (x, u, 1.0, torch.ones(2, device=dev)), (x, u.cpu()), (torch.zeros(1, 720897, device=dev), u[:1])):
        with pytest.raises(RuntimeError):
            sampling.sample(*args)


# --------------------------------------------------------------------------- launch counts
def _kernels_and_count(fn):
    """Nodes of the CUDA graph that `fn` captures, and what it counted."""
    import ctypes
    from hetero_cp_ringattn_b200.utils import launches
    fn()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with launches.capture() as cap:
        with torch.cuda.graph(graph):
            fn()
    n = ctypes.c_size_t()
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value, cap.launches


@pytest.mark.parametrize("tokens,units", [(0, 1), (1, 1), (3, 1), (4, 1), (8, 1), (11, 1), (12, 1), (16, 1), (16, 0), (47, 4), (48, 4)])
def test_append_counts_what_it_launches(dev, tokens, units):
    k, v, ks, vs = _strided_cache(4, 1, 16, 64, "e4m3", dev)
    cos, sin = (t.to(dev) for t in ref.rope_cos_sin(torch.arange(64), 64, 10000.0))
    x = torch.randn(tokens, 3 * 64, device=dev)
    pos = torch.arange(tokens, dtype=torch.int32, device=dev)
    unit = torch.tensor([[0, 16 * i, min(16, tokens - 16 * i), 16 * i] if 16 * i < tokens else [-1, 0, 0, 0] for i in range(units)],
                        dtype=torch.int32, device=dev).view(units, 4)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    nodes, counted = _kernels_and_count(lambda: paged.rope_append_kv8(x, cos, sin, pos, unit, table, k, v, ks, vs, heads=1))
    assert counted == nodes == (0 if tokens == 0 else 2 if 0 < 12 * units <= tokens else 1)


@pytest.mark.parametrize("n", [0, 1, 5])
def test_other_operators_count_what_they_launch(dev, n):
    k, v, ks, vs = _strided_cache(2, 1, 16, 64, "int8", dev)
    table = torch.zeros(max(n, 1), 1, dtype=torch.int32, device=dev)
    q = torch.randn(n, 2, 64, device=dev).bfloat16()
    lens, cu = torch.ones(max(n, 1), dtype=torch.int32, device=dev), torch.arange(max(n, 1) + 1, dtype=torch.int32, device=dev)
    cu *= n > 0
    x, u = torch.randn(n, 100, device=dev), torch.rand(n, device=dev)
    for fn in (lambda: paged.attention_kv8(q, k, v, ks, vs, table, lens, cu), lambda: paged.gather_kv8(k, v, ks, vs, table[0], n),
               lambda: sampling.sample(x, u)):
        nodes, counted = _kernels_and_count(fn)
        assert nodes == counted


# --------------------------------------------------------------------------- the decoder
@pytest.mark.parametrize("code,page,rows", [("e4m3", 64, 3), ("int8", 16, 10)])
def test_decoder_on_the_gpu_matches_the_quantised_oracle(dev, code, page, rows):
    """Prompts in pieces and batched graph steps against the float32 oracle with quantised K and V. bf16
    activations err as in the engine's tests (0.15 / 0.025 of the logits' scale at most / on average);
    they also move K and V across rounding boundaries of their codes, which doubles the room."""
    from hetero_cp_ringattn_b200.models.paged import PagedDecoder
    from hetero_cp_ringattn_b200.models.weights import ModelWeights, PreparedWeights
    from test_paged_cpu import _oracle
    cfg = preset("tiny-gpu")
    cfg.attention_bias = True
    hf = ModelWeights.random_init(cfg, seed=3, device=dev, dtype=torch.bfloat16)
    dec = PagedDecoder(cfg, PreparedWeights.from_weights(hf), rows=rows, max_context=512, kv_cache=code, page=page)
    host = ModelWeights(cfg, {n: t.cpu() for n, t in hf.tensors.items()})
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, cfg.vocab_size, (20 + 37 * (r % 5),), generator=g) for r in range(rows)]

    def close(got, r):
        want = _oracle(host, seqs[r], page, code)
        err, scale = (got.float().cpu() - want).abs(), max(1.0, float(want.std()))
        assert err.max() < 0.3 * scale and err.mean() < 0.05 * scale, (r, float(err.max()), float(err.mean()))

    for r in range(rows):
        close(dec.prefill(r, seqs[r], piece=2 * page), r)
    active = [r for r in range(rows) if r != 1]
    for _ in range(3):
        nxt = torch.randint(0, cfg.vocab_size, (len(active),), generator=g)
        out = dec.step(active, nxt.to(dev))
        for j, r in enumerate(active):
            seqs[r] = torch.cat([seqs[r], nxt[j:j + 1]])
        for j in (0, len(active) - 1):
            close(dec.last_logits[j], active[j])
        assert torch.equal(out, dec.last_logits.float().argmax(-1))
    dec.check_device()
    want = [0 if r == 1 else len(seqs[r]) for r in range(rows)]
    want[1] = len(seqs[1])
    assert dec.cache.kv_len.tolist() == want == dec.cache.lens


@pytest.mark.parametrize("graphs", [True, False])
def test_decoder_raises_for_what_kernels_reported(dev, graphs):
    """A token id past the vocabulary, given to a step, a prompt and generate: raised by the next call once the
    device has run, or by check_device and generate, once each, and the decoder goes on."""
    from hetero_cp_ringattn_b200.errors import KernelError
    from hetero_cp_ringattn_b200.models.paged import PagedDecoder
    from hetero_cp_ringattn_b200.models.weights import PreparedWeights
    cfg = preset("tiny-gpu")
    dec = PagedDecoder(cfg, PreparedWeights.random(cfg, seed=0, device=dev), rows=2, max_context=128, use_graphs=graphs)
    prompt, bad = torch.arange(9), torch.tensor([cfg.vocab_size])
    want = dec.generate([prompt], 4)[0]
    dec.prefill(0, prompt)
    for call in (lambda: dec.step([0], bad), lambda: dec.prefill(1, bad)):
        for after in (lambda: dec.step([0], want[:1]), lambda: dec.prefill(1, prompt), dec.check_device):
            call()
            torch.cuda.synchronize()
            lens = list(dec.cache.lens)
            with pytest.raises(KernelError, match="301"):
                after()
            assert dec.cache.lens == lens
            dec.check_device()
    for r in (0, 1):
        dec.release(r)
    with pytest.raises(KernelError, match="301"):
        dec.generate([bad], 2)
    assert torch.equal(dec.generate([prompt], 4)[0], want)


def test_decoder_capture_survives_a_garbage_collection(dev, monkeypatch):
    """Another decoder with a captured graph becomes unreachable, in a cycle, while a step is captured, and
    the collector is due at every allocation."""
    import gc
    from hetero_cp_ringattn_b200.models.paged import PagedDecoder
    from hetero_cp_ringattn_b200.models.weights import PreparedWeights
    cfg = preset("tiny-gpu")
    w = PreparedWeights.random(cfg, seed=0, device=dev)
    prompt = torch.arange(9)
    old = [PagedDecoder(cfg, w, rows=1, max_context=64)]
    want = old[0].generate([prompt], 6)[0]
    new = PagedDecoder(cfg, w, rows=1, max_context=64)
    new.prefill(0, prompt)
    first = want[:1]
    append = paged.rope_append_kv8

    def drop(*a, **k):
        if old:
            cycle = [old.pop()]
            cycle.append(cycle)
            del cycle
        [[i] for i in range(100)]
        return append(*a, **k)

    monkeypatch.setattr(paged, "rope_append_kv8", drop)
    was = gc.get_threshold()
    gc.set_threshold(1, 1, 1)
    try:
        got = [first]
        for _ in range(5):
            got.append(new.step([0], got[-1]).clone())
    finally:
        gc.set_threshold(*was)
    assert not old and torch.equal(torch.cat(got), want)


@pytest.mark.parametrize("graphs", [True, False])
def test_decoder_results_of_a_step_stay(dev, graphs):
    from hetero_cp_ringattn_b200.models.paged import PagedDecoder
    from hetero_cp_ringattn_b200.models.weights import PreparedWeights
    from test_paged_cpu import check_results_stay
    cfg = preset("tiny-gpu")
    check_results_stay(PagedDecoder(cfg, PreparedWeights.random(cfg, seed=0, device=dev), rows=2, max_context=64, use_graphs=graphs))


def test_decoder_graph_equals_eager_and_is_reproducible(dev):
    from hetero_cp_ringattn_b200.models.paged import PagedDecoder
    from hetero_cp_ringattn_b200.models.weights import PreparedWeights
    cfg = preset("tiny-gpu")
    w = PreparedWeights.random(cfg, seed=0, device=dev)
    prompts = [torch.arange(n) % cfg.vocab_size for n in (5, 130, 64)]
    runs = []
    for graphs in (True, False, True):
        dec = PagedDecoder(cfg, w, rows=4, max_context=256, use_graphs=graphs)
        runs.append(dec.generate(prompts, 12, temperature=0.8, top_k=50, top_p=0.95, seed=9))
        dec.check_device()
        assert dec.cache.lens == [0] * 4 and int(dec.cache.counters[1] - dec.cache.counters[0]) == dec.cache.pages
    for a in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], a))
