"""Plain PyTorch oracles of the paged 8-bit KV cache ops (`paged.py`), row by row.

They are what CPU tensors run and what the kernels are tested against; none is on the GPU hot path.
"""

from __future__ import annotations

from typing import Optional

import torch

from ..errors import RingError

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
MIN_EXP, MAX_EXP = -40, 40


def pow2_scale(amax: torch.Tensor, code: torch.dtype) -> torch.Tensor:
    """The smallest power of two s in [2^-40, 2^40] with amax <= QMAX * s."""
    m, e = torch.frexp(amax.clamp(max=2.0 ** 100))
    limit, sub = (0.875, 9) if code == torch.float8_e4m3fn else (0.9921875, 7)
    e = torch.where(m <= limit, e - sub, e - sub + 1).clamp(MIN_EXP, MAX_EXP)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)))


def encode(x: torch.Tensor, code: torch.dtype) -> torch.Tensor:
    """Codes of x (already divided by the scale): nearest, ties to even, saturated; NaN stays NaN in
    e4m3 and becomes 0 in int8."""
    if code == torch.float8_e4m3fn:
        return x.clamp(-448.0, 448.0).to(code)
    return torch.nan_to_num(x.round().clamp(-127.0, 127.0), nan=0.0).to(code)


def plan_step(add, kv_len, block_table, ring, counters, page: int, max_tokens: int, out) -> None:
    n, old = [int(x) for x in add], [int(x) for x in kv_len]
    rows, width = block_table.shape
    head, tail = int(counters[0]), int(counters[1])
    size = ring.numel()
    have = [-(-o // page) for o in old]
    need = [max(0, -(-(o + max(a, 0)) // page) - h) for a, o, h in zip(n, old, have)]
    back = [h if a < 0 else 0 for a, h in zip(n, have)]
    grow = [max(a, 0) for a in n]
    status = 0
    if sum(grow) > max_tokens:
        status = 3
    elif any(h + x > width for h, x in zip(have, need)):
        status = 2
    elif sum(need) > min(max(tail - head, 0), size) + sum(back):
        status = 1
    elif min(max(tail - head, 0), size) + sum(back) > size:
        status = 4
    out.row.fill_(-1)
    out.pos.zero_()
    out.slot.fill_(-1)
    out.unit.zero_()
    out.unit[:, 0] = -1
    new_len, t, u = list(old), 0, 0
    cu = [0] * (rows + 1)
    taken = 0
    if status == 0:
        released = [int(block_table[r, j]) for r in range(rows) for j in range(back[r])]
        for i, page_id in enumerate(released):
            ring[(tail + i) % size] = page_id
        for r in range(rows):
            cu[r] = t
            if n[r] < 0:
                new_len[r] = 0
                continue
            for j in range(need[r]):
                block_table[r, have[r] + j] = ring[(head + taken) % size]
                taken += 1
            p, end = old[r], old[r] + grow[r]
            new_len[r] = end
            while p < end:
                m = min(end, (p // page + 1) * page) - p
                out.unit[u] = torch.tensor([r, t, m, p], dtype=torch.int32)
                first = int(block_table[r, p // page]) * page + p % page
                out.row[t:t + m] = r
                out.pos[t:t + m] = torch.arange(p, p + m, dtype=torch.int32)
                out.slot[t:t + m] = torch.arange(first, first + m)
                u, t, p = u + 1, t + m, p + m
        cu[rows] = t
        tail += len(released)
    out.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    out.kv_len.copy_(torch.tensor(new_len, dtype=torch.int32))
    out.counters.copy_(torch.tensor([head + taken, tail]))
    out.info.copy_(torch.tensor([t, u, taken, status], dtype=torch.int32))


def _store(x, unit, block_table, data, scale) -> None:
    """Rows x [tokens, kv_heads, D] (float32) into the units' blocks."""
    P, code = data.shape[2], data.dtype
    for r, t0, m, p0 in unit.tolist():
        if r < 0:
            continue
        page, start = int(block_table[r, p0 // P]), p0 % P
        new = x[t0:t0 + m]
        amax = torch.nan_to_num(new.abs(), nan=0.0).amax(dim=(0, 2))
        s = pow2_scale(amax, code)
        if start:
            old = scale[page].clone()
            s = torch.maximum(old, s)
            f = (old / s).view(-1, 1, 1)
            stored = data[page, :, :start].float()
            again = encode(stored * f, code)
            data[page, :, :start] = torch.where(f < 1, again.float(), stored).to(code)
        scale[page] = s
        data[page, :, start:start + m] = encode(new / s.view(1, -1, 1), code).transpose(0, 1)


def _check_places(unit, block_table, pages: int, P: int, tokens: int, pos, positions: int) -> None:
    """Raise for what the kernel reports to its status word, before anything is written."""
    if tokens and not 0 <= int(pos.min()) <= int(pos.max()) < positions:
        raise RingError(f"a position outside the rotary tables' {positions}")
    rows, width = block_table.shape
    for r, t0, m, p0 in unit.tolist():
        if r < 0:
            continue
        ok = r < rows and t0 >= 0 and 1 <= m <= tokens - t0 and p0 >= 0 and p0 % P + m <= P and p0 // P < width
        if not ok or p0 + m > positions or not 0 <= int(block_table[r, p0 // P]) < pages:
            raise RingError(f"unit {(r, t0, m, p0)} is out of range")


def rope_append_kv8(qkv, cos, sin, pos, unit, block_table, k, v, k_scale, v_scale, heads: int,
                    q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    T, Hkv, D = qkv.shape[0], k.shape[1], k.shape[3]
    if qkv.shape[1] != (heads + 2 * Hkv) * D:
        raise RingError("qkv must have heads + 2 kv_heads heads a row")
    _check_places(unit, block_table, k.shape[0], k.shape[2], T, pos[:T], cos.shape[0])
    x = qkv.float().view(T, heads + 2 * Hkv, D)
    c, s = cos[pos[:T].long()].unsqueeze(1), sin[pos[:T].long()].unsqueeze(1)
    x1, x2 = x[:, :heads + Hkv, : D // 2], x[:, :heads + Hkv, D // 2:]
    rot = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
    _store(rot[:, heads:], unit, block_table, k, k_scale)
    _store(x[:, heads + Hkv:], unit, block_table, v, v_scale)
    if q_out is None:
        q_out = torch.empty(T, heads, D, dtype=torch.bfloat16 if qkv.dtype == torch.float32 else qkv.dtype)
    q_out.copy_(rot[:, :heads].view(q_out.shape))
    return q_out


def cached_rows(data, scale, table_row, n: int, dtype=torch.float32) -> torch.Tensor:
    """The values of the first n cached rows, [n, kv_heads, D]."""
    P = data.shape[2]
    pages = table_row[: -(-n // P)].long()
    if len(pages) and not 0 <= int(pages.min()) <= int(pages.max()) < data.shape[0]:
        raise RingError(f"a page id outside the pool of {data.shape[0]} pages")   # (the kernels report and read zeros)
    raw = data.view(torch.uint8)[pages].view(data.dtype)
    x = raw.to(torch.float32).to(dtype) * scale[pages].to(dtype).view(len(pages), data.shape[1], 1, 1)
    return x.transpose(1, 2).reshape(-1, data.shape[1], data.shape[3])[:n]


def attention_kv8(q, k, v, k_scale, v_scale, block_table, kv_len, cu, scale: float, out=None, want_lse: bool = True,
                  dtype=torch.float32):
    """Also the kernel tests' oracle (`dtype` float64)."""
    T, H, D = q.shape
    Hkv = k.shape[1]
    o = torch.zeros(T, H, D, dtype=dtype, device=q.device)
    lse = torch.full((H, T), float("-inf"), dtype=dtype, device=q.device)
    bounds = list(range(kv_len.numel() + 1)) if cu is None else cu.tolist()
    for b, n in enumerate(kv_len.tolist()):
        t0, t1 = bounds[b], bounds[b + 1]
        for i, t in enumerate(range(t0, t1)):
            seen = n - (t1 - t0) + i + 1
            if seen <= 0:
                continue
            kk = cached_rows(k, k_scale, block_table[b], seen, dtype).repeat_interleave(H // Hkv, dim=1)
            vv = cached_rows(v, v_scale, block_table[b], seen, dtype).repeat_interleave(H // Hkv, dim=1)
            s = torch.einsum("hd,nhd->hn", q[t].to(dtype), kk) * scale
            lse[:, t] = torch.logsumexp(s, dim=-1)
            o[t] = torch.einsum("hn,nhd->hd", torch.softmax(s, dim=-1), vv)
    if dtype != torch.float32:
        return o, lse
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    out.copy_(o.view(out.shape))
    return out, (lse if want_lse else None)


def gather_kv8(k, v, k_scale, v_scale, table_row, n: int, out):
    for data, scale, o in ((k, k_scale, out[0]), (v, v_scale, out[1])):
        o[:, :n] = cached_rows(data, scale, table_row, n).transpose(0, 1).to(o.dtype)
    return out
