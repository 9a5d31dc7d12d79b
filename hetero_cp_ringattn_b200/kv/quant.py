"""The paged 8-bit KV cache of one rank: every layer's pages and scales, and the page bookkeeping on
the device (block tables, lengths, free-page ring), grown and released by `ops.paged.plan_step`.

Half the bytes of the bf16 arena (`kv/arena.py`) per cached token, one float32 scale per (page, KV
head) for K and V beside them. Lengths and tables live on the GPU, so a decode step needs no host
round trip; the host keeps a mirror of the lengths and of the number of free pages, which raises a
`CapacityError` before a step that does not fit is launched.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from ..errors import CapacityError, RingError
from ..ops import paged

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Kv8Cache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, rows: int, max_context: int,
                 pages: Optional[int] = None, page: int = 64, code: str = "e4m3", device=None):
        if code not in CODES:
            raise RingError(f"unknown 8-bit KV cache type {code!r}; known: {sorted(CODES)}")
        if page not in (16, 32, 64, 128):
            raise CapacityError(f"8-bit KV cache page of {page} tokens: 16, 32, 64 or 128")
        if head_dim not in (64, 128):
            raise RingError(f"8-bit KV cache head_dim {head_dim}: 64 or 128")
        if rows < 1 or rows > 1024:
            raise CapacityError(f"8-bit KV cache of {rows} rows: 1 to 1024")
        self.rows, self.page, self.code = int(rows), int(page), code
        self.max_context = int(max_context)
        width = -(-self.max_context // page)
        self.pages = int(pages if pages is not None else rows * width)
        shape = (layers, self.pages, kv_heads, page, head_dim)
        dev = torch.device(device or "cpu")
        # zeroed: a page's unwritten tail is finite (the kernels mask it in any case)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=dev).view(CODES[code])
        self.v = torch.zeros(shape, dtype=torch.uint8, device=dev).view(CODES[code])
        self.k_scale = torch.ones(shape[:3], dtype=torch.float32, device=dev)
        self.v_scale = torch.ones(shape[:3], dtype=torch.float32, device=dev)
        self.block_table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        self.kv_len = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.ring = torch.arange(self.pages, dtype=torch.int32, device=dev)
        self.counters = torch.tensor([0, self.pages], dtype=torch.int64, device=dev)
        self.lens = [0] * rows           # host mirror
        self.free_pages = self.pages

    @property
    def bytes(self) -> int:
        """Bytes of the codes and scales."""
        return 2 * self.k.numel() + 4 * 2 * self.k_scale.numel()

    def layer(self, i: int):
        """(k, v, k_scale, v_scale) of layer i."""
        return self.k[i], self.v[i], self.k_scale[i], self.v_scale[i]

    def after(self, add: Sequence[int]) -> Tuple[List[int], int]:
        """The host mirror (lengths, free pages) after a step of add[r] tokens for row r, negative to release
        it; changes nothing. Raises `CapacityError` where the device plan would not fit."""
        if len(add) != self.rows:
            raise RingError(f"{len(add)} entries for {self.rows} rows")
        held = lambda n: -(-n // self.page)  # noqa: E731
        new = [0 if a < 0 else n + a for a, n in zip(add, self.lens)]
        for r, n in enumerate(new):
            if n > self.max_context:
                raise CapacityError(f"row {r}: {n} tokens exceed the context capacity {self.max_context}")
        free = self.free_pages + sum(held(n) for n in self.lens) - sum(held(n) for n in new)
        if free < 0:
            raise CapacityError(f"8-bit KV cache: {-free} pages short ({self.pages} in all)")
        return new, free

    def commit(self, state: Tuple[List[int], int]) -> None:
        """Take over what `after` returned. Belongs directly behind the launch of the step's plan, so that the
        mirror never counts tokens that the device was not told about."""
        self.lens, self.free_pages = state

    def reserve(self, add: Sequence[int]) -> List[int]:
        """Check and account for a step in one go, for callers that launch its plan next."""
        self.commit(self.after(add))
        return [int(a) for a in add]

    def plan(self, add: torch.Tensor, max_tokens: int, out: Optional[paged.StepPlan] = None) -> paged.StepPlan:
        """The device's side of a reserved step; lengths and counters are updated in place."""
        if out is None:
            out = paged.StepPlan.empty(self.rows, self.page, max_tokens, self.kv_len.device, kv_len=self.kv_len,
                                       counters=self.counters)
        return paged.plan_step(add, self.kv_len, self.block_table, self.ring, self.counters, page=self.page,
                               max_tokens=max_tokens, out=out)

    def release(self, row: int) -> None:
        if not 0 <= row < self.rows:
            raise RingError(f"row {row}: the cache has {self.rows}")
        add = [0] * self.rows
        add[row] = -1
        state = self.after(add)
        self.plan(torch.tensor(add, dtype=torch.int32, device=self.kv_len.device), 1)
        self.commit(state)
