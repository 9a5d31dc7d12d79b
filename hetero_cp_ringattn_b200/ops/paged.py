"""Front-ends of the paged 8-bit KV cache: the step plan (block tables and slot maps from request
lengths), the rotary append, attention over the cache, and the gather back to bf16.

A layer's cache is `k`, `v` [pages, kv_heads, page, head_dim] in 8 bits (float8_e4m3fn or int8; page
16, 32, 64 or 128 tokens, head_dim 64 or 128) with float32 scales `k_scale`, `v_scale` [pages, kv_heads]:
a code c stands for c * scale. `rope_append_kv8` makes the scales powers of two, so rescaling an open
block is an exponent shift and code * scale is exact in bf16; the readers take any positive scale from
2^-60 to 2^60. `kv.quant.Kv8Cache` holds the tensors of every layer with the page bookkeeping.

CUDA tensors go to the native kernels on the current stream (outputs and workspace come from the
caching allocator of that stream, nothing is kept between calls); CPU tensors to the oracles in
`paged_reference.py`. All calls can be captured in a CUDA graph: lengths and tables are read on the
device, no call synchronises.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Optional, Tuple

import torch

from . import paged_reference as pref
from ._ext import native
from ..utils import launches


@dataclasses.dataclass
class StepPlan:
    """One step's bookkeeping on the device. Tokens are numbered row by row: row r's new tokens are
    cu[r] .. cu[r + 1] - 1. Entries past the step's tokens (units) hold -1 in `row` and `slot`
    (`unit`'s first column)."""
    cu: torch.Tensor          # int32 [rows + 1]
    row: torch.Tensor         # int32 [max_tokens] row of each token
    pos: torch.Tensor         # int32 [max_tokens] its position in the row
    slot: torch.Tensor        # int64 [max_tokens] page id * page + offset
    unit: torch.Tensor        # int32 [units, 4] touched blocks: row, first token, tokens, first position
    kv_len: torch.Tensor      # int32 [rows] rows after the step
    counters: torch.Tensor    # int64 [2] head and tail of the page ring after the step
    info: torch.Tensor        # int32 [4] tokens, units, pages taken, status (PLAN_STATUS)

    @classmethod
    def empty(cls, rows: int, page: int, max_tokens: int, device, kv_len: Optional[torch.Tensor] = None,
              counters: Optional[torch.Tensor] = None) -> "StepPlan":
        """Buffers for steps of up to `max_tokens` new tokens. Given `kv_len` / `counters`, the plan
        updates these tensors in place."""
        i32 = dict(dtype=torch.int32, device=device)
        return cls(cu=torch.empty(rows + 1, **i32), row=torch.empty(max_tokens, **i32),
                   pos=torch.empty(max_tokens, **i32),
                   slot=torch.empty(max_tokens, dtype=torch.int64, device=device),
                   unit=torch.empty(max_units(rows, page, max_tokens), 4, **i32),
                   kv_len=kv_len if kv_len is not None else torch.empty(rows, **i32),
                   counters=counters if counters is not None else torch.empty(2, dtype=torch.int64, device=device),
                   info=torch.empty(4, **i32))


PLAN_STATUS = {0: "ok", 1: "not enough free pages", 2: "a row outgrows its block table", 3: "more tokens than the plan holds",
               4: "more pages given back than the ring has places for"}


def max_units(rows: int, page: int, max_tokens: int) -> int:
    """Blocks that `max_tokens` new tokens in `rows` rows can touch at most."""
    return min(max_tokens, max_tokens // page + 2 * rows)


def plan_step(add: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor, ring: torch.Tensor,
              counters: torch.Tensor, *, page: int, max_tokens: int, out: Optional[StepPlan] = None) -> StepPlan:
    """Grow row r by add[r] >= 0 tokens, or release it (add[r] < 0), and build the step's slot map.

    `kv_len` int32 [rows] lengths; `block_table` int32 [rows, width]; `ring` int32 [pages], a FIFO of
    free page ids whose entries counters[0] .. counters[1] - 1 (int64, modulo the ring's size) are free.
    New pages are taken in row order, first from the ring, then from rows released in this same step;
    released pages join the ring's end in row order (the free and the released pages of a step together must
    not exceed the ring's size: it holds every page of the pool). `block_table` and `ring` are updated in place (new
    entries only), the new lengths and counters go to the plan. A step that does not fit changes nothing
    and sets info[3] (PLAN_STATUS). At most 4096 rows."""
    if out is None:
        out = StepPlan.empty(add.shape[0], page, max_tokens, add.device)
    if not add.is_cuda:
        pref.plan_step(add, kv_len, block_table, ring, counters, page, max_tokens, out)
        return out
    native().plan_step(add, kv_len, block_table, ring, counters, page, out.cu, out.row, out.pos, out.slot,
                       out.unit, out.kv_len, out.counters, out.info)
    launches.count()
    return out


def rope_append_kv8(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor,
                    unit: torch.Tensor, block_table: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, *, heads: int,
                    q_out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q and k of every token at pos[t] (rotate-half, tables `cos` / `sin` [positions, D / 2]),
    write q out and code k and v into the rows' blocks.

    `qkv` [tokens, (heads + 2 kv_heads) * D] in float32, bf16 or f16; `pos`, `unit` of the step's plan
    (`plan_step`, or the same lists made elsewhere; entries with row -1 are skipped). Whole blocks are stored
    from 12 tokens an entry of `unit` on, so a prompt's list should not be much longer than its blocks: pass
    the part in use. Block scales: a new block's follows from its new
    tokens, an open block's grows with them (its stored codes are rescaled). Returns q [tokens, heads, D]
    in `q_out`'s type (default: qkv's, bf16 for float32). A token whose position lies outside the rotary
    tables gets q = 0, and a unit whose row, tokens, positions or page id are out of range stores nothing;
    both are reported to `status`, an int32 [>= 4] error word (on the CPU they raise and nothing is written)."""
    if not qkv.is_cuda:
        return pref.rope_append_kv8(qkv, cos, sin, pos, unit, block_table, k, v, k_scale, v_scale, heads, q_out)
    q, launched = native().rope_append_kv8(qkv, cos, sin, pos, unit, block_table, k, v, k_scale, v_scale, heads, q_out,
                                           status)
    launches.count(launched)
    return q


def attention_kv8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
                  cu: Optional[torch.Tensor] = None, *, max_q: int = 1, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, want_lse: bool = True,
                  status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of q [tokens, heads, D] (bf16 or f16) over the requests' cached rows.

    Request b has the query tokens cu[b] .. cu[b + 1] - 1 (None: token b) and kv_len[b] cached rows; its
    query token i of m sees rows 0 .. kv_len[b] - m + i. `max_q` is the most query tokens that a request
    has: the tiles' shape goes by it, the results do not (a request with more is right, but slower). `cu`
    past the tokens of q and page ids outside the pool (read as zeros) are reported to `status`; on the CPU
    they raise. Returns (o [tokens, heads, D], lse [heads, tokens] natural
    log, or None); a token that sees no row gets o = 0, lse = -inf, so the partials of several ranks' shards
    merge like the other attention's (`reference.merge_partials`). At most 1024 requests a call. Meant for
    decode steps and short segments (drafts to verify): for a long segment read the rows back with
    `gather_kv8` and use `kernels.attention`."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if not q.is_cuda:
        return pref.attention_kv8(q, k, v, k_scale, v_scale, block_table, kv_len, cu, scale, out, want_lse)
    o, lse = native().attention_kv8(q, k, v, k_scale, v_scale, block_table, kv_len, cu, max_q, scale, out,
                                    want_lse, status)
    launches.count(2 if q.shape[0] else 0)
    return o, (lse if want_lse else None)


def gather_kv8(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               block_table_row: torch.Tensor, n: int,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first n cached rows of one request as bf16 K and V [kv_heads, n or more, D] in position order,
    what `kernels.attention` reads. `out`: buffers to write into. Rows of a page id outside the pool are
    zeros (on the CPU they raise)."""
    if not k.is_cuda:
        if out is None:
            out = tuple(torch.empty(k.shape[1], n, k.shape[3], dtype=torch.bfloat16) for _ in "kv")
        return pref.gather_kv8(k, v, k_scale, v_scale, block_table_row, n, out)
    out = native().gather_kv8(k, v, k_scale, v_scale, block_table_row, n, *(out or (None, None)))
    launches.count(1 if n else 0)
    return out
