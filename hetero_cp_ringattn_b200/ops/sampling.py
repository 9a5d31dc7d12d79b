"""Batched sampling with temperature, top-k, top-p and min-p from given uniform numbers.

For a row of logits l with maximum L and temperature T > 0 every token has the distance
d = (L - l) / T and the fixed-point weight w = floor(2^31 exp(-d)). Tokens are ordered by (d, index):
top-k keeps the first k; top-p keeps, of those, the tokens whose exclusive cumulative weight lies below
max(1, floor(top_p * total)); min-p keeps w >= floor(2^31 min_p). The token is the first one in
vocabulary order whose inclusive cumulative kept weight exceeds floor(u * kept total). The weights come
from a fixed sequence of rounded float32 operations and the rest is integer arithmetic, so the same
logits, settings and numbers give the same token on the CPU and on the GPU, in any batch.
"""

from __future__ import annotations

import math
from typing import Optional, Union

import torch

from ._ext import native
from ..errors import RingError
from ..utils import launches

# Taylor coefficients of 2^g, highest power first: the polynomial of the kernel, operation by operation
_EXP2 = [math.log(2.0) ** i / math.factorial(i) for i in range(7, -1, -1)]
_LOG2E = 1.4426950408889634
# the largest float32 below 1: numbers from 1 on and NaN count as it, as in the kernel
_U_MAX = 1.0 - 2.0 ** -24

Setting = Union[float, int, torch.Tensor]


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
           top_p: Setting = 1.0, min_p: Setting = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token id (int64) per row of `logits` [rows, vocab] (float32 or bf16; a GPU row holds at most
    720896 tokens). `u` float32 [rows] in [0, 1) (below: 0; from 1 on, or NaN:
    the largest number below 1). Each setting is a number or one value per row (float32;
    top_k int32). temperature <= 0: the lowest index of the maximum. Off: top_k <= 0, top_p outside (0, 1),
    min_p <= 0. NaN logits count as -inf; a row without any other gives -1."""
    if not logits.is_cuda:
        return _sample_host(logits, u, temperature, top_k, top_p, min_p, out)
    t = (temperature, 0.0) if isinstance(temperature, torch.Tensor) else (None, temperature)
    k = (top_k, 0) if isinstance(top_k, torch.Tensor) else (None, top_k)
    p = (top_p, 0.0) if isinstance(top_p, torch.Tensor) else (None, top_p)
    m = (min_p, 0.0) if isinstance(min_p, torch.Tensor) else (None, min_p)
    token = native().sample(logits, u, *t, *k, *p, *m, out)
    launches.count(1 if logits.shape[0] else 0)
    return token


def weights(d: torch.Tensor) -> torch.Tensor:
    """floor(2^31 exp(-d)) as int64 for float32 d in [0, 64]."""
    y = d * _LOG2E
    n = y.round()
    g = n - y
    w = torch.full_like(g, _EXP2[0])
    for c in _EXP2[1:]:
        w = w * g + c
    return (w * 2147483648.0).to(torch.int64) >> n.to(torch.int64)


def _share(total: int, x: float) -> int:
    """floor(total * x), x in [0, 1] held in 24 bits."""
    q = max(0, min(int(x * 16777216.0), 1 << 24)) if x == x else 0
    return (total * q) >> 24


def _sample_host(logits, u, temperature, top_k, top_p, min_p, out) -> torch.Tensor:
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise RingError("logits must be float32 or bfloat16 [rows, vocab]")
    rows = logits.shape[0]
    if u.shape != (rows,):
        raise RingError("u must have one number per row")
    pick = lambda s, b: s[b].item() if isinstance(s, torch.Tensor) else s  # noqa: E731
    if out is None:
        out = torch.empty(rows, dtype=torch.int64)
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    for b in range(rows):
        x = logits[b].float()
        x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
        top = x.max()
        T, k, p, m = f32(pick(temperature, b)), int(pick(top_k, b)), f32(pick(top_p, b)), f32(pick(min_p, b))
        if float(top) == float("-inf"):
            out[b] = -1
            continue
        if not float(T) > 0:
            out[b] = int((x == top).to(torch.int8).argmax())
            continue
        d = torch.where(x == top, torch.zeros_like(x), (top - x) / T)
        d = torch.where(torch.isnan(d), torch.full_like(d, 64.0), d.clamp(max=64.0))
        w = weights(d)
        order = torch.sort(d, stable=True).indices
        ws = w[order]
        if k > 0:
            ws[k:] = 0
        if 0.0 < float(p) < 1.0:
            cum = torch.cumsum(ws, 0)
            ws = torch.where(cum - ws < max(1, _share(int(cum[-1]), float(p))), ws, torch.zeros_like(ws))
        if float(m) > 0:
            ws = torch.where(ws >= int(min(float(m), 1.0) * 2147483648.0), ws, torch.zeros_like(ws))
        kept = torch.zeros_like(w)
        kept[order] = ws
        cum = torch.cumsum(kept, 0)
        r = float(u[b])
        target = _share(int(cum[-1]), r if r < _U_MAX else _U_MAX)
        out[b] = int(torch.searchsorted(cum, torch.tensor([target]), right=True))
    return out
