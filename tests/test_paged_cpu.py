"""The paged 8-bit KV cache, its step plan and the batched sampler on the CPU: the oracles that the
kernels are tested against, and the single-rank decoder built on them."""

import gc
import json
import math
import random
import weakref

import pytest
import torch

from hetero_cp_ringattn_b200.config import preset
from hetero_cp_ringattn_b200.errors import CapacityError, KernelError, RingError
from hetero_cp_ringattn_b200.kv.quant import CODES, Kv8Cache
from hetero_cp_ringattn_b200.models.paged import PagedDecoder
from hetero_cp_ringattn_b200.models.weights import ModelWeights, PreparedWeights
from hetero_cp_ringattn_b200.ops import paged, paged_reference as pref, reference as ref, sampling


# --------------------------------------------------------------------------- step plan
@pytest.mark.parametrize("page", [1, 3, 16])
def test_plan_random_walk_keeps_every_page_owned_once(page):
    """Rows grow and are released at random; after every step the pages of all rows and the free part
    of the ring are each page exactly once, and the slot map agrees with the tables."""
    r = random.Random(page)
    rows, width = 5, 7
    pages = rows * width - 6
    kv_len = torch.zeros(rows, dtype=torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    ring = torch.randperm(pages).to(torch.int32)
    counters = torch.tensor([0, pages])
    lens = [0] * rows
    for _ in range(200):
        add = [r.choice([-1, 0, 1, 1, 2, r.randrange(0, 2 * page + 2)]) for _ in range(rows)]
        p = paged.plan_step(torch.tensor(add, dtype=torch.int32), kv_len, table, ring, counters, page=page, max_tokens=8 * page)
        held = lambda n: -(-n // page)  # noqa: E731
        new = [0 if a < 0 else n + a for a, n in zip(add, lens)]
        free = int(counters[1] - counters[0])
        ok = (sum(max(a, 0) for a in add) <= 8 * page and all(held(n) <= width for n in new) and
              free + sum(held(n) for n in lens) - sum(held(n) for n in new) >= 0)
        assert (int(p.info[3]) == 0) == ok
        if not ok:
            assert p.kv_len.tolist() == lens and torch.equal(p.counters, counters) and int(p.info[0]) == 0
            assert (p.slot == -1).all() and (p.unit[:, 0] == -1).all()
            continue
        lens, kv_len, counters = new, p.kv_len, p.counters
        assert kv_len.tolist() == lens
        n = int(counters[1] - counters[0])
        owned = [int(table[i, j]) for i in range(rows) for j in range(held(lens[i]))]
        owned += [int(ring[(int(counters[0]) + i) % pages]) for i in range(n)]
        assert sorted(owned) == list(range(pages))
        total = int(p.info[0])
        assert total == sum(max(a, 0) for a in add) and (p.row[total:] == -1).all() and (p.slot[total:] == -1).all()
        covered = 0
        for t in range(total):
            i, pos = int(p.row[t]), int(p.pos[t])
            assert int(p.cu[i]) <= t < int(p.cu[i + 1]) and pos == lens[i] - int(p.cu[i + 1]) + t
            assert int(p.slot[t]) == int(table[i, pos // page]) * page + pos % page
        for i, t0, m, p0 in p.unit[: int(p.info[1])].tolist():
            assert p0 // page == (p0 + m - 1) // page and int(p.row[t0]) == i and int(p.pos[t0]) == p0
            covered += m
        assert covered == total


@pytest.mark.parametrize("add,status", [([17, 0, 0], 1), ([0, 33, 0], 2), ([16, 16, 16], 3), ([16, -1, 0], 0)])
def test_plan_refuses_what_does_not_fit(add, status):
    """Pages of 8 tokens: 1 free page (row 1's 2 more once it is released), rows of at most 4 pages, a plan of 40 tokens."""
    kv_len = torch.tensor([8, 15, 0], dtype=torch.int32)
    table = torch.tensor([[3, -1, -1, -1], [0, 1, -1, -1], [-1] * 4], dtype=torch.int32)
    ring = torch.tensor([9, 2, 9, 9], dtype=torch.int32)
    p = paged.plan_step(torch.tensor(add, dtype=torch.int32), kv_len, table, ring, torch.tensor([5, 6]), page=8, max_tokens=40)
    assert int(p.info[3]) == status
    if status:
        assert p.kv_len.tolist() == [8, 15, 0] and p.counters.tolist() == [5, 6] and (p.slot == -1).all()
    else:
        assert p.kv_len.tolist() == [24, 0, 0] and table[0].tolist() == [3, 2, 0, -1] and p.counters.tolist() == [7, 8]


def _crowded_ring(free):
    """Row 0 holds 3 pages, row 1 one, and the ring has 4 places, `free` of them taken: releasing row 0 fits
    up to one free page."""
    kv_len = torch.tensor([40, 16], dtype=torch.int32)
    table = torch.tensor([[5, 6, 7], [8, -1, -1]], dtype=torch.int32)
    return kv_len, table, torch.tensor([0, 1, 2, 3], dtype=torch.int32), torch.tensor([7, 7 + free])


@pytest.mark.parametrize("free,status", [(0, 0), (1, 0), (2, 4), (4, 4), (9, 4)])
def test_plan_gives_back_no_more_pages_than_the_ring_holds(free, status):
    kv_len, table, ring, counters = _crowded_ring(free)
    p = paged.plan_step(torch.tensor([-1, 0], dtype=torch.int32), kv_len, table, ring, counters, page=16, max_tokens=4)
    assert int(p.info[3]) == status and status in paged.PLAN_STATUS
    if status:
        assert ring.tolist() == [0, 1, 2, 3] and p.kv_len.tolist() == [40, 16] and p.counters.tolist() == [7, 7 + free]
    else:
        want = [0, 1, 2, 3]
        for i, page_id in enumerate((5, 6, 7)):
            want[(7 + free + i) % 4] = page_id
        assert ring.tolist() == want and p.kv_len.tolist() == [0, 16] and p.counters.tolist() == [7, 10 + free]


def test_cache_mirror_and_capacity_errors():
    c = Kv8Cache(1, 2, 64, rows=2, max_context=100, page=16, pages=6)
    c.plan(torch.tensor(c.reserve([50, 17]), dtype=torch.int32), 67)
    assert c.lens == [50, 17] and c.free_pages == 0 and c.kv_len.tolist() == [50, 17]
    with pytest.raises(CapacityError):
        c.reserve([0, 16])              # no page left
    with pytest.raises(CapacityError):
        c.reserve([51, 0])              # past the context
    assert c.lens == [50, 17]
    c.release(0)
    assert c.free_pages == 4 and c.kv_len.tolist() == [0, 17]
    c.plan(torch.tensor(c.reserve([0, 16]), dtype=torch.int32), 16)
    for bad in (dict(code="e5m2"), dict(page=48), dict(rows=0)):
        with pytest.raises(RingError):
            Kv8Cache(1, 2, 64, **{**dict(rows=2, max_context=64, page=16), **bad})
    with pytest.raises(RingError):
        Kv8Cache(1, 2, 96, rows=1, max_context=64)


# --------------------------------------------------------------------------- append
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_values_are_within_a_code_step(code):
    """Tokens written in several pieces of growing size into open blocks: every cached value is within
    one rounding of its own size (e4m3: 2^-4 relative, or half the smallest step 2^-9 s, twice after
    rescaling; int8: half a step, at most one after rescaling) of the rotated input."""
    torch.manual_seed(0)
    H, Hkv, D, P, T = 2, 2, 64, 16, 45
    c = Kv8Cache(1, Hkv, D, rows=1, max_context=64, page=P, code=code)
    cos, sin = ref.rope_cos_sin(torch.arange(64), D, 10000.0)
    x = torch.randn(T, (H + 2 * Hkv) * D) * torch.linspace(0.01, 3.0, T).unsqueeze(1)
    x[7] = 0.0
    at = 0
    for n in (1, 1, 5, 20, 3, 15):
        plan = c.plan(torch.tensor(c.reserve([n]), dtype=torch.int32), n)
        q = paged.rope_append_kv8(x[at:at + n], cos, sin, plan.pos, plan.unit, c.block_table, *c.layer(0), heads=H)
        want = ref.apply_rope(x[at:at + n, :H * D].view(n, H, D), torch.arange(at, at + n), 10000.0)
        assert torch.equal(q, want.to(torch.bfloat16))
        at += n
    assert at == T
    k, v, ks, vs = c.layer(0)
    want_k = ref.apply_rope(x[:, H * D:(H + Hkv) * D].view(T, Hkv, D), torch.arange(T), 10000.0)
    for data, scale, want in ((k, ks, want_k), (v, vs, x[:, (H + Hkv) * D:].view(T, Hkv, D))):
        got = pref.cached_rows(data, scale, c.block_table[0], T)
        s = scale[c.block_table[0][torch.arange(T) // P].long()].unsqueeze(-1)
        assert torch.equal(torch.frexp(scale)[0], torch.full_like(scale, 0.5))       # powers of two
        step = torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -9) if code == "e4m3" else s.expand_as(want)
        assert ((got - want).abs() <= step * 1.0001).all()


@pytest.mark.parametrize("unit,table,pos", [
    ([0, 0, 2, 7], [1], [7, 8]), ([0, 0, 2, 7], [1], [6, 7]), ([0, 0, 2, 0], [1], [-1, 0]), ([0, 0, 2, -1], [1], [0, 1]),
    ([0, 0, 2, 0], [-1], [0, 1]), ([0, 0, 2, 0], [2], [0, 1]), ([1, 0, 2, 0], [1], [0, 1]), ([0, 1, 2, 0], [1], [0, 1]),
    ([0, 0, 2, 16], [1], [0, 1])])
def test_append_refuses_places_out_of_range(unit, table, pos):
    """Positions past and before the rotary tables (of 8 positions, pages of 16), page ids, rows and tokens
    that are not there: refused, with nothing written."""
    c = Kv8Cache(1, 1, 64, rows=1, max_context=16, page=16, pages=2)
    cos, sin = ref.rope_cos_sin(torch.arange(8), 64, 10000.0)
    i32 = dict(dtype=torch.int32)
    with pytest.raises(RingError):
        paged.rope_append_kv8(torch.randn(2, 3 * 64), cos, sin, torch.tensor(pos, **i32), torch.tensor([unit], **i32),
                              torch.tensor([table], **i32), *c.layer(0), heads=1)
    assert not c.k.view(torch.uint8).any() and not c.v.view(torch.uint8).any()
    assert (c.k_scale == 1).all() and (c.v_scale == 1).all()


def test_scale_is_the_smallest_power_of_two_that_holds_the_maximum():
    for code, top in ((torch.float8_e4m3fn, 448.0), (torch.int8, 127.0)):
        a = torch.cat([torch.tensor([top, top * 1.0001, top * 0.5, 1e-30, 0.0, 1e30]), torch.rand(1000) * 1000])
        s = pref.pow2_scale(a, code)
        inside = (s > 2.0 ** -40) & (s < 2.0 ** 40)
        assert (a[inside] <= top * s[inside]).all() and (a[inside] > top * s[inside] / 2).all()
        assert s[3] == s[4] == 2.0 ** -40 and s[5] == 2.0 ** 40


def test_gather_of_no_rows():
    c = Kv8Cache(1, 2, 64, rows=1, max_context=48, page=16)
    out = tuple(torch.full((2, 3, 64), 7.0, dtype=torch.bfloat16) for _ in "kv")
    for k, v in (paged.gather_kv8(*c.layer(0), c.block_table[0], 0), paged.gather_kv8(*c.layer(0), c.block_table[0], 0, out=out)):
        assert k.shape == v.shape and (k == 7).all() and (v == 7).all()


@pytest.mark.parametrize("bad", [-1, 3])
def test_readers_refuse_page_ids_outside_the_pool(bad):
    c = Kv8Cache(1, 1, 64, rows=1, max_context=48, page=16, pages=3)
    k, v, ks, vs = c.layer(0)
    q, lens = torch.randn(1, 2, 64), lambda n: torch.tensor([n], dtype=torch.int32)
    for row, n, ok in (([0, 2, bad], 33, False), ([0, bad, 1], 20, False), ([0, 2, bad], 32, True), ([bad, bad, bad], 0, True)):
        table = torch.tensor([row], dtype=torch.int32)
        for call in (lambda: paged.attention_kv8(q, k, v, ks, vs, table, lens(n)), lambda: paged.gather_kv8(k, v, ks, vs, table[0], n)):
            if ok:
                call()
            else:
                with pytest.raises(RingError, match="page id"):
                    call()
    with pytest.raises((RingError, IndexError)):
        paged.attention_kv8(q, k, v, ks, vs, torch.tensor([[0, 1, 2]], dtype=torch.int32), lens(3), torch.tensor([0, 2]))


# --------------------------------------------------------------------------- sampling
def _naive(logits, u, T, k, p, m):
    """The definition by float64 weights and an explicit loop."""
    x = logits.double()
    w = torch.exp((x - x.max()) / T)
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i))
    keep = order[:k] if k > 0 else order
    if 0 < p < 1:
        total, cum, cut = float(sum(w[i] for i in keep)), 0.0, []
        for i in keep:
            if cut and cum >= p * total:
                break
            cut.append(i)
            cum += float(w[i])
        keep = cut
    keep = sorted(i for i in keep if w[i] >= m)
    total, cum = float(sum(w[i] for i in keep)), 0.0
    for i in keep:
        cum += float(w[i])
        if cum > u * total:
            return i
    return keep[-1]


@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.1),
                                      (0.9, 20, 0.9, 0.02)])
def test_sample_matches_the_definition(settings):
    torch.manual_seed(1)
    logits = torch.randn(40, 200) * 3
    u = torch.rand(40)
    got = sampling.sample(logits, u, *settings).tolist()
    assert got == [_naive(logits[b], float(u[b]), *settings) for b in range(40)]


def test_sample_edge_rows():
    ninf = float("-inf")
    logits = torch.tensor([[1.0, 3.0, 3.0, 0.0], [ninf] * 4, [ninf, ninf, -5.0, ninf], [float("nan"), 1.0, float("nan"), ninf],
                           [float("inf"), 0.0, float("inf"), 5.0], [torch.finfo(torch.float32).min] * 4])
    u = torch.tensor([0.99, 0.5, 0.5, 0.5, 0.9, 0.6])
    assert sampling.sample(logits, u, 0.0).tolist() == [1, -1, 2, 1, 0, 0]          # greedy: the lowest index
    assert sampling.sample(logits, u, 1.0, top_k=1).tolist() == [1, -1, 2, 1, 0, 0]
    # row 0 has the cumulative weights e^-2, 1 + e^-2, 2 + e^-2, 2 + e^-2 + e^-3: 0.977 of the total at
    # token 2; equal logits share the draw of rows 4 and 5
    assert sampling.sample(logits, u, 1.0).tolist() == [3, -1, 2, 1, 2, 2]
    assert sampling.sample(logits, u, 1e-30).tolist() == [2, -1, 2, 1, 2, 2]
    assert sampling.sample(logits, u, torch.full((6,), 1.0), torch.full((6,), 2, dtype=torch.int32), 1.0, 1.0).tolist() == \
        [2, -1, 2, 1, 2, 1]
    with pytest.raises(RingError):
        sampling.sample(logits[0], u)
    with pytest.raises(RingError):
        sampling.sample(logits, u[:3])


@pytest.mark.parametrize("u", [1.0 - 2.0 ** -24, 1.0, 2.0, float("nan")])
def test_sample_largest_uniform_number(u):
    """The second token's weight 2^31 e^-16.23 = 192 is 1.5 times 2^-24 of the total S: u = 1 - 2^-24, the largest
    float32 below 1, reaches floor(S - S 2^-24), past the first token; one unit of 2^-24 less does not."""
    logits = torch.tensor([[0.0, -16.23]])
    w = sampling.weights(torch.tensor([0.0, 16.23])).tolist()
    assert w[0] == 2 ** 31 and 130 < w[1] < 250
    assert sampling.sample(logits, torch.tensor([u])).tolist() == [1]
    assert sampling.sample(logits, torch.tensor([1.0 - 2.0 ** -23])).tolist() == [0]


def test_weights_follow_exp():
    d = torch.linspace(0, 20, 4001)
    w = sampling.weights(d).double() / 2.0 ** 31
    want = torch.exp(-d.double())
    # the argument d log2(e) is rounded once (2^-24 relative: d 2^-24 of the result), eight roundings
    # of the polynomial, and the floor at 2^-31
    assert ((w - want).abs() <= want * (d.double() * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -31).all()


# --------------------------------------------------------------------------- the decoder
def _quantised(x, page, code):
    """Rows [n, heads, D] as an append of them all leaves them: per (block, head) one power-of-two scale."""
    top = 448.0 if code == "e4m3" else 127.0
    out = torch.empty_like(x)
    for b in range(0, x.shape[0], page):
        blk = x[b:b + page]
        s = 2.0 ** torch.ceil(torch.log2(blk.abs().amax((0, 2), keepdim=True).double() / top)).float()
        out[b:b + page] = pref.encode(blk / s, CODES[code]).float() * s
    return out


def _oracle(hf, ids, page, code):
    """Float32 forward of the model with every layer's K and V quantised; the last token's logits."""
    cfg = hf.cfg
    H, Hkv, D, L = cfg.num_heads, cfg.kv_heads, cfg.head_dim, len(ids)
    t = lambda n: hf[n].float()  # noqa: E731
    pos = torch.arange(L)
    x = t("model.embed_tokens.weight")[ids]
    for i in range(cfg.num_layers):
        p = f"model.layers.{i}."
        h = ref.rmsnorm(x, t(p + "input_layernorm.weight"), cfg.rms_norm_eps)
        q, k, v = (ref.linear(h, t(p + f"self_attn.{n}_proj.weight"), t(p + f"self_attn.{n}_proj.bias") if cfg.attention_bias
                              else None).view(L, -1, D) for n in "qkv")
        q, k = (ref.apply_rope(y, pos, cfg.rope_theta, cfg.rope_scaling) for y in (q, k))
        o, _ = ref.full_attention(q, _quantised(k, page, code), _quantised(v, page, code), pos, pos)
        x = x + ref.linear(o.reshape(L, H * D), t(p + "self_attn.o_proj.weight"))
        h = ref.rmsnorm(x, t(p + "post_attention_layernorm.weight"), cfg.rms_norm_eps)
        x = x + ref.linear(ref.swiglu(ref.linear(h, t(p + "mlp.gate_proj.weight")), ref.linear(h, t(p + "mlp.up_proj.weight"))),
                           t(p + "mlp.down_proj.weight"))
    return ref.linear(ref.rmsnorm(x[-1:], t("model.norm.weight"), cfg.rms_norm_eps), hf.lm_head().float())[0]


def _model(bias=False):
    cfg = preset("tiny-gpu")
    cfg.attention_bias = bias
    return ModelWeights.random_init(cfg, seed=5, dtype=torch.float32, std=0.05)


@pytest.mark.parametrize("code,page,bias", [("e4m3", 16, False), ("int8", 32, True)])
def test_decoder_matches_the_quantised_oracle(code, page, bias):
    """Two rows of different lengths, prompts in pieces, three batched steps with given tokens. The
    decoder's K and V differ from the oracle's by float32 summation order alone, which now and then
    moves a value across a rounding boundary of its code: one code step of one element, 2^-3 of it, in
    a head dim of 64 and a context of dozens, about 1e-3 of the logits' spread; 2e-2 allowed."""
    hf = _model(bias)
    dec = PagedDecoder(hf.cfg, PreparedWeights.from_weights(hf, dtype=torch.float32), rows=3, max_context=128, kv_cache=code,
                       page=page, device=torch.device("cpu"))
    g = torch.Generator().manual_seed(2)
    seqs = {0: torch.randint(0, hf.cfg.vocab_size, (37,), generator=g), 2: torch.randint(0, hf.cfg.vocab_size, (16,), generator=g)}
    for r, ids in seqs.items():
        got = dec.prefill(r, ids, piece=2 * page)
        want = _oracle(hf, ids, page, code)
        assert (got - want).abs().max() < 2e-2 * want.std()
    for _ in range(3):
        nxt = torch.randint(0, hf.cfg.vocab_size, (2,), generator=g)
        out = dec.step([0, 2], nxt)
        for j, r in enumerate((0, 2)):
            seqs[r] = torch.cat([seqs[r], nxt[j:j + 1]])
            want = _oracle(hf, seqs[r], page, code)
            assert (dec.last_logits[j] - want).abs().max() < 2e-2 * want.std()
            assert int(out[j]) == int(dec.last_logits[j].argmax())
    assert dec.cache.lens == [40, 0, 19]
    with pytest.raises(RingError):
        dec.step([2, 0], nxt)
    with pytest.raises(CapacityError):
        dec.prefill(1, torch.zeros(129, dtype=torch.int64))


def _small_decoder(**kw):
    hf = _model()
    kw = {**dict(rows=3, max_context=64, page=16, device=torch.device("cpu")), **kw}
    return PagedDecoder(hf.cfg, PreparedWeights.from_weights(hf, dtype=torch.float32), **kw)


def test_refused_steps_and_prompts_change_nothing(monkeypatch):
    """Whatever a call raises for, the host's lengths stay the device's, and the next step is as if the call
    had not been made."""
    dec, ref_dec = _small_decoder(), _small_decoder()
    for d in (dec, ref_dec):
        d.prefill(0, torch.arange(9))
        d.prefill(2, torch.arange(5))
    one = lambda n, v=1.0: torch.full((n,), v)  # noqa: E731
    for kw in (dict(tokens=torch.arange(3)), dict(tokens=torch.arange(1)), dict(u=one(3)), dict(u=one(1)), dict(temperature=one(3)),
               dict(top_k=one(1).int()), dict(top_p=one(4)), dict(min_p=one(1))):
        with pytest.raises(RingError):
            dec.step([0, 2], **{**dict(tokens=torch.arange(2), u=one(2, 0.5), temperature=1.0), **kw})
    for row, ids, piece in ((-1, torch.arange(3), 16), (3, torch.arange(3), 16), (1, torch.arange(3), 0), (1, torch.arange(65), 16),
                            (1, torch.arange(0), 16)):
        with pytest.raises(RingError):
            dec.prefill(row, ids, piece)
    for row in (-1, 3):
        with pytest.raises(RingError):
            dec.release(row)
    # a failure on the way to the plan
    with monkeypatch.context() as m:
        m.setattr(paged, "plan_step", lambda *a, **k: (_ for _ in ()).throw(MemoryError()))
        for call in (lambda: dec.step([0, 2], torch.arange(2)), lambda: dec.prefill(1, torch.arange(20)), lambda: dec.release(0)):
            with pytest.raises(MemoryError):
                call()
            assert dec.cache.lens == dec.cache.kv_len.tolist() == [9, 0, 5]
    # and behind it: the tokens are in the cache on both sides
    with monkeypatch.context() as m:
        m.setattr(sampling, "sample", lambda *a, **k: (_ for _ in ()).throw(MemoryError()))
        for d in (dec, ref_dec):
            with pytest.raises(MemoryError):
                d.step([0], torch.arange(1))
            assert d.cache.lens == d.cache.kv_len.tolist() == [10, 0, 5]
    free = dec.cache.pages - sum(-(-n // 16) for n in dec.cache.lens)
    assert dec.cache.free_pages == free == int(dec.cache.counters[1] - dec.cache.counters[0])
    assert torch.equal(dec.step([0, 2], torch.arange(2)), ref_dec.step([0, 2], torch.arange(2)))
    assert torch.equal(dec.last_logits, ref_dec.last_logits)
    number = torch.tensor(0.7)                     # a setting as a tensor of one number is for every row
    assert torch.equal(dec.step([0, 2], torch.arange(2), one(2, 0.5), number), ref_dec.step([0, 2], torch.arange(2), one(2, 0.5), 0.7))


def test_step_with_a_temperature_needs_uniform_numbers():
    """Without u no earlier step's numbers are drawn with; greedy steps need none."""
    dec = _small_decoder()
    for r in (0, 1):
        dec.prefill(r, torch.arange(4))
    dec.step([0, 1], torch.arange(2), torch.tensor([0.9, 0.9]), temperature=1.0)
    for t in (1.0, torch.tensor([0.0, 0.5]), torch.tensor(2.0)):
        with pytest.raises(RingError, match="needs u"):
            dec.step([0, 1], torch.arange(2), temperature=t)
    assert dec.cache.lens == [5, 5, 0]
    for t in (0.0, -1.0, float("nan"), torch.zeros(2)):
        assert torch.equal(dec.step([0, 1], torch.arange(2), temperature=t), dec.last_logits.argmax(-1))


def test_decoder_is_freed_without_a_garbage_collection():
    dec = _small_decoder()
    dec.generate([torch.arange(5)] * 2, 3)
    gone = weakref.ref(dec)
    gc.collect()
    gc.disable()
    try:
        del dec
        assert gone() is None
    finally:
        gc.enable()


def test_generate_raises_for_a_report_and_clears_it():
    """The status word as a kernel would leave it (the CPU forms have none of their own)."""
    dec = _small_decoder()
    want = dec.generate([torch.arange(5)], 3)[0]
    dec.status = torch.tensor([18, 402, 7, 0, 0, 0, 0, 0], dtype=torch.int32)
    with pytest.raises(KernelError, match="402"):
        dec.generate([torch.arange(5)], 3)
    assert not dec.status.any() and dec.cache.lens == [0, 0, 0]
    assert torch.equal(dec.generate([torch.arange(5)], 3)[0], want)


def test_prefill_attention_has_an_error_word_of_its_own(monkeypatch):
    """A report of another kernel (a token id, a position) must not end the waits of the prefill attention."""
    from hetero_cp_ringattn_b200.models import paged as model
    dec = _small_decoder()
    dec.status = torch.zeros(16, dtype=torch.int32)
    words = {"append": [], "attention": []}

    def spy(name, fn):
        def call(*a, status=None, **k):
            words[name].append(status.data_ptr())
            return fn(*a, **k)
        return call

    monkeypatch.setattr(paged, "rope_append_kv8", spy("append", paged.rope_append_kv8))
    monkeypatch.setattr(model.K, "attention", spy("attention", model.K.attention))
    dec.prefill(0, torch.arange(20), piece=16)
    assert len(words["append"]) == len(words["attention"]) == 2 * dec.cfg.num_layers
    assert len(set(words["append"])) == len(set(words["attention"])) == 1
    assert abs(words["append"][0] - words["attention"][0]) >= 16
    for i in (0, 8):
        dec.status[i] = 16
        with pytest.raises(KernelError):
            dec.check_device()
        dec.check_device()


def test_generate_leaves_rows_in_use_alone():
    """A session in row 0: prompts take other rows, and are refused where those do not suffice."""
    dec, alone = _small_decoder(), _small_decoder()
    for d in (dec, alone):
        d.prefill(0, torch.arange(20))
    prompts = [torch.arange(5), torch.arange(30, 41)]
    got = dec.generate(prompts, 4, temperature=0.9, seed=1)
    want = _small_decoder().generate(prompts, 4, temperature=0.9, seed=1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert dec.cache.lens == [20, 0, 0]
    with pytest.raises(RingError, match="2 free rows"):
        dec.generate(prompts + prompts, 4)
    assert torch.equal(dec.step([0], torch.tensor([3])), alone.step([0], torch.tensor([3])))
    assert torch.equal(dec.last_logits, alone.last_logits)


def check_results_stay(dec):
    """Tokens and logits of a step do not change with later steps of the same size."""
    vocab = dec.cfg.vocab_size
    for r in (0, 1):
        dec.prefill(r, torch.arange(4 + r))
    kept = []
    for i in range(4):
        out = dec.step([0, 1], torch.tensor([11 * i + 1, 7 * i + 300]) % vocab)
        kept.append((out, out.tolist(), dec.last_logits, dec.last_logits.tolist()))
    assert len({tuple(k[1]) for k in kept}) > 1
    for out, values, logits, logit_values in kept:
        assert out.tolist() == values and logits.tolist() == logit_values


def test_results_of_a_step_stay():
    check_results_stay(_small_decoder())


@pytest.mark.parametrize("had,n", [(0, 1), (0, 16), (0, 17), (5, 11), (5, 12), (15, 2), (16, 40), (20, 64)])
def test_prompt_hands_the_append_its_own_units(monkeypatch, had, n):
    """However many rows the cache has: exactly the blocks that the piece touches, all of its tokens."""
    dec = _small_decoder(rows=40, max_context=128)
    if had:
        dec.prefill(3, torch.arange(had))
    append, seen = paged.rope_append_kv8, []

    def spy(qkv, cos, sin, pos, unit, *a, **k):
        seen.append(unit.tolist())
        return append(qkv, cos, sin, pos, unit, *a, **k)

    monkeypatch.setattr(paged, "rope_append_kv8", spy)
    dec.prefill(3, torch.arange(n))
    assert len(seen) == dec.cfg.num_layers
    for units in seen:
        assert [u[3] // 16 for u in units] == list(range(had // 16, (had + n - 1) // 16 + 1))
        assert all(u[0] == 3 for u in units) and sum(u[2] for u in units) == n


def test_prompt_that_fails_between_pieces_keeps_the_mirror(monkeypatch):
    dec = _small_decoder()
    piece, calls = dec._piece, []

    def twice(*a):
        calls.append(a)
        if len(calls) > 1:
            raise MemoryError()
        return piece(*a)

    monkeypatch.setattr(dec, "_piece", twice)
    with pytest.raises(MemoryError):
        dec.prefill(1, torch.arange(40), piece=16)
    assert dec.cache.lens == dec.cache.kv_len.tolist() == [0, 16, 0]
    dec.release(1)
    assert dec.cache.free_pages == dec.cache.pages == int(dec.cache.counters[1] - dec.cache.counters[0])


def test_decoder_generate_is_reproducible_and_releases_its_pages():
    hf = _model()
    dec = PagedDecoder(hf.cfg, PreparedWeights.from_weights(hf, dtype=torch.float32), rows=2, max_context=64, device=torch.device("cpu"))
    prompts = [torch.arange(9), torch.arange(20)]
    a = dec.generate(prompts, 5, temperature=0.9, top_k=30, top_p=0.95, min_p=0.01, seed=3)
    b = dec.generate(prompts, 5, temperature=0.9, top_k=30, top_p=0.95, min_p=0.01, seed=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[0].shape == (5,)
    assert dec.cache.free_pages == dec.cache.pages and dec.cache.lens == [0, 0]
    one = dec.generate(prompts[1:], 5)[0]
    assert torch.equal(one, dec.generate(prompts, 5)[1])        # a row does not depend on its batch
    with pytest.raises(RingError):
        dec.generate([prompts[0]] * 3, 2)


def test_infer_on_the_8bit_cache(capsys):
    from hetero_cp_ringattn_b200.cli import main
    assert main(["infer", "--model-preset", "tiny-gpu", "--device", "cpu", "--prompt", "ring", "--max-tokens", "4",
                 "--max-context", "64", "--kv-cache", "int8", "--kv-page", "16", "--top-k", "8", "--temperature", "0.7"]) == 0
    out = json.loads(capsys.readouterr().out)
    assert len(out["tokens"]) == 4 and out["kv_cache"] == "int8" and out["kv_bytes"] > 0
    assert math.isfinite(sum(out["tokens"]))


_INFER = ["infer", "--model-preset", "tiny-gpu", "--device", "cpu", "--prompt", "ring", "--max-tokens", "3", "--max-context", "64"]


@pytest.mark.parametrize("extra", [["--top-k", "1", "--temperature", "5"], ["--min-p", "0.2"], ["--kv-page", "16"],
                                   ["--kv-cache", "int8", "--num-domains", "2"], ["--kv-cache", "e4m3", "--ratio", "5:5:1"],
                                   ["--kv-cache", "int8", "--chunk-sizes", "1,1"]])
def test_infer_refuses_flags_it_would_not_follow(extra):
    """The 8-bit cache's sampling and page flags without it, and layouts of several ranks with it."""
    from hetero_cp_ringattn_b200.cli import main
    with pytest.raises((SystemExit, RingError), match="needs --kv-cache|WORLD_SIZE|for 1 domains"):
        main(_INFER + extra)


def test_infer_on_the_8bit_cache_with_one_domain(capsys):
    from hetero_cp_ringattn_b200.cli import main
    outs = []
    for extra in ([], ["--num-domains", "1", "--ratio", "5", "--kv-page", "64"]):
        assert main(_INFER + ["--kv-cache", "int8"] + extra) == 0
        outs.append(json.loads(capsys.readouterr().out))
    assert outs[0] == outs[1]
