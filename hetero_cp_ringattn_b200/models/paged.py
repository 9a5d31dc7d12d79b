"""Single-rank decoder over the paged 8-bit KV cache: prompts in pieces, batched decode steps, and
sampling on the device.

One decode step is plan -> per layer [QKV projection, rotary append, attention, output projection,
MLP] -> LM head -> sample, captured in a CUDA graph per power of two of active rows (lengths, block
tables, sampling settings and uniform numbers are read on the device, so a graph serves any set of
rows; tokens past the active rows belong to no request and cost next to nothing). A prompt piece appends its rows to the cache, reads the row back as bf16
(`gather_kv8`) and runs the tcgen05 prefill attention on it, so a prompt sees the same quantised K
and V whether it came in one piece or several (pieces of whole pages).

Several ranks keep the bf16 arena (`models/llama.py`).
"""

from __future__ import annotations

import gc
import math
import weakref
from typing import Dict, List, Optional, Sequence

import torch

from ..config import ModelConfig
from ..errors import KernelError, RingError
from ..kv.quant import Kv8Cache
from ..ops import kernels as K
from ..ops import paged
from ..ops import reference as ref
from ..ops import sampling
from ..utils import launches
from .weights import PreparedWeights

GEMV_ROWS = 8      # decode batches up to here run the streaming GEMVs, larger ones the GEMM


class PagedDecoder:
    def __init__(self, cfg: ModelConfig, weights: PreparedWeights, *, rows: int = 8, max_context: int = 8192,
                 kv_cache: str = "e4m3", page: int = 64, pages: Optional[int] = None,
                 device: Optional[torch.device] = None, use_graphs: bool = True):
        cfg.validate()
        self.cfg, self.w = cfg, weights
        self.device = device or weights.embed.device
        self.cuda = self.device.type == "cuda"
        self.H, self.Hkv, self.D = cfg.num_heads, cfg.kv_heads, cfg.head_dim
        self.scale = 1.0 / math.sqrt(self.D)
        self.cache = Kv8Cache(cfg.num_layers, self.Hkv, self.D, rows=rows, max_context=max_context, pages=pages,
                              page=page, code=kv_cache, device=self.device)
        cos, sin = ref.rope_cos_sin(torch.arange(max_context, device=self.device), self.D, cfg.rope_theta,
                                    scaling=cfg.rope_scaling)
        self.cos, self.sin = cos.contiguous(), sin.contiguous()
        self.act = torch.bfloat16 if self.cuda else torch.float32
        # the kernels' error words (see `_word`), and their copy on the host, brought there behind every step
        # and prompt
        self.status = torch.zeros(16, dtype=torch.int32, device=self.device) if self.cuda else None
        self._seen = torch.zeros(16, dtype=torch.int32, pin_memory=True) if self.cuda else None
        self.use_graphs = use_graphs and self.cuda
        self._steps: Dict[int, "_Step"] = {}
        self._logits_now: Optional[torch.Tensor] = None   # the last step's, in its buffer

    # ------------------------------------------------------------------ prompts
    @torch.no_grad()
    def prefill(self, row: int, ids: torch.Tensor, piece: int = 8192) -> torch.Tensor:
        """Append a prompt (or a session's next segment) to `row`, at most `piece` tokens at a time;
        returns the last token's logits [vocab], float32. A prompt that does not fit is refused whole; one
        that fails on the way leaves the row with the pieces that were appended."""
        self._raise_seen()
        if not 0 <= row < self.cache.rows:
            raise RingError(f"row {row}: the cache has {self.cache.rows}")
        if ids.numel() < 1:
            raise RingError("empty prompt")
        if piece < 1:
            raise RingError(f"pieces of {piece} tokens")
        add = [0] * self.cache.rows
        add[row] = int(ids.numel())
        had = self.cache.lens[row]
        self.cache.after(add)
        ids = ids.reshape(-1).to(self.device).int()
        x = None
        for at in range(0, ids.numel(), piece):
            x = self._piece(row, ids[at:at + piece], had + at)
        self._look()
        return self._logits(x[-1:])[0].float()

    def _piece(self, row: int, ids: torch.Tensor, had: int) -> torch.Tensor:
        w, cfg, c = self.w, self.cfg, self.cache
        T, L = ids.numel(), had + ids.numel()
        add = [0] * c.rows
        add[row] = T
        state = c.after(add)
        plan = c.plan(torch.tensor(add, dtype=torch.int32, device=self.device), T)
        c.commit(state)
        # the blocks that this row's tokens touch: the plan's list has room for units of every row, and the
        # append's launch goes by the list's length
        unit = plan.unit[:-(-L // c.page) - had // c.page]
        pos = torch.arange(had, L, dtype=torch.int32, device=self.device)
        x = K.embedding(ids, w.embed, status=self._word(0)) if self.cuda else w.embed[ids.long()].float()
        back = [torch.empty(self.Hkv, L, self.D, dtype=torch.bfloat16, device=self.device) for _ in "kv"]
        for li, lw in enumerate(w.layers):
            xn = K.rmsnorm(x, lw.in_norm, cfg.rms_norm_eps)
            qkv = K.gemm(xn, lw.wqkv, "bias" if lw.bqkv is not None else "store", bias=lw.bqkv)
            q = paged.rope_append_kv8(qkv, self.cos, self.sin, plan.pos, unit, c.block_table, *c.layer(li),
                                      heads=self.H, q_out=torch.empty(T, self.H, self.D, dtype=self.act, device=self.device),
                                      status=self._word(0))
            k, v = paged.gather_kv8(*c.layer(li), c.block_table[row], L, out=tuple(back))
            o, _ = K.attention(q, k, v, pos, L, scale=self.scale, want_lse=False, status=self._word(1))
            x = K.gemm(o.reshape(T, -1), lw.wo, "residual", residual=x)
            g = K.gemm(K.rmsnorm(x, lw.post_norm, cfg.rms_norm_eps), lw.wgu, "swiglu")
            x = K.gemm(g, lw.wd, "residual", residual=x)
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        """LM head of hidden rows [n, hidden]: float32 up to 8 rows, else the activations' type."""
        n = x.shape[0]
        if n <= GEMV_ROWS:
            out = torch.empty(n, self.cfg.vocab_size, dtype=torch.float32, device=self.device)
            return K.gemv(x, self.w.lm_head, "f32", y_f32=out, norm_w=self.w.final_norm, eps=self.cfg.rms_norm_eps)
        return K.gemm(K.rmsnorm(x, self.w.final_norm, self.cfg.rms_norm_eps), self.w.lm_head, "store")

    # ------------------------------------------------------------------ decode
    @torch.no_grad()
    def step(self, rows: Sequence[int], tokens: torch.Tensor, u: Optional[torch.Tensor] = None,
             temperature=0.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
        """One decode step: rows[i] (ascending) takes tokens[i] and gets its next token, int64
        [len(rows)] on the device. Settings are numbers or one value per row; `u` the uniform
        numbers (needed when any temperature is positive). `last_logits` are the step's logits."""
        self._raise_seen()
        rows = [int(r) for r in rows]
        n = len(rows)
        if n == 0 or any(b <= a for a, b in zip(rows, rows[1:])) or rows[0] < 0 or rows[-1] >= self.cache.rows:
            raise RingError("rows must be ascending row numbers of the cache")
        add = [0] * self.cache.rows
        for r in rows:
            add[r] = 1
        for name, x in (("tokens", tokens), ("u", u), ("temperature", temperature), ("top_k", top_k), ("top_p", top_p),
                        ("min_p", min_p)):
            single = x is not tokens and x is not u and isinstance(x, torch.Tensor) and x.dim() == 0   # a number
            if isinstance(x, torch.Tensor) and not single and x.numel() != n:
                raise RingError(f"{name}: {x.numel()} values for {n} rows")
        if u is None and (bool((temperature > 0).any()) if isinstance(temperature, torch.Tensor) else temperature > 0):
            raise RingError("a positive temperature needs u")
        state = self.cache.after(add)
        bucket = 1 << (n - 1).bit_length()
        st = self._steps.get(bucket)
        if st is None:
            st = self._steps[bucket] = _Step(self, bucket)
        out = st.run(n, add, state, tokens, u, temperature, top_k, top_p, min_p)
        self._look()
        return out

    @property
    def last_logits(self) -> Optional[torch.Tensor]:
        """A copy of the last step's logits [rows, vocab], which the next step may overwrite."""
        return None if self._logits_now is None else self._logits_now.clone()

    def release(self, row: int) -> None:
        """Give the row's pages back."""
        self.cache.release(row)

    def check_device(self) -> None:
        """Wait for the device and raise if a kernel reported an error since the last one raised for (a token,
        page id or position out of range). `generate` ends with it; `prefill` and `step` raise, without
        waiting, for what earlier ones are known to have reported."""
        word = [] if self.status is None else self.status.tolist()
        if any(word[::8]):
            self.status.zero_()          # each report is raised once, and says nothing about later calls
            if self._seen is not None:
                self._seen.zero_()       # (its copies are done: the read above waited for them)
            raise KernelError(f"device status {word}")

    def _word(self, i: int) -> Optional[torch.Tensor]:
        """Error word 0, for the kernels that report bad places and go on, or 1, for the prefill attention: it
        gives up its waits, with copies in flight, once its word is set, so only its own reports may set it."""
        return None if self.status is None else self.status[8 * i:8 * i + 8]

    def _look(self) -> None:
        if self._seen is not None:
            self._seen.copy_(self.status, non_blocking=True)

    def _raise_seen(self) -> None:
        if self._seen is not None and any(self._seen[::8].tolist()):
            self.check_device()

    @torch.no_grad()
    def generate(self, prompts: Sequence[torch.Tensor], max_new_tokens: int, *, temperature=0.0, top_k=0, top_p=1.0,
                 min_p=0.0, seed: int = 0, piece: int = 8192) -> List[torch.Tensor]:
        """Generate for several prompts at once, each in a row that holds nothing yet and is released at the
        end; the ids per prompt, on the device."""
        rows = [r for r, n in enumerate(self.cache.lens) if n == 0][:len(prompts)]
        if len(prompts) > len(rows):
            raise RingError(f"{len(prompts)} prompts for {len(rows)} free rows")
        gen = torch.Generator(device=self.device).manual_seed(seed)
        settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        logits, started = [], []
        try:
            for r, p in zip(rows, prompts):
                started.append(r)
                logits.append(self.prefill(r, p, piece))
            draw = lambda: torch.rand(len(rows), generator=gen, device=self.device)  # noqa: E731
            cur = sampling.sample(torch.stack(logits), draw(), **settings)
            outs = [cur]
            for _ in range(max_new_tokens - 1):
                cur = self.step(rows, cur, draw(), **settings)
                outs.append(cur)
            self.check_device()
        finally:
            for r in started:
                self.release(r)
        return list(torch.stack(outs, 1))


class _Step:
    """Static buffers of a step of up to `n` active rows, and the captured step."""

    def __init__(self, dec: PagedDecoder, n: int):
        # (no cycle: a decoder that is given up frees its cache and graphs at once)
        self.d, self.n = weakref.proxy(dec), n
        dev, c = dec.device, dec.cache
        self.add = torch.zeros(c.rows, dtype=torch.int32, device=dev)
        self.tokens = torch.zeros(n, dtype=torch.int32, device=dev)
        self.u = torch.zeros(n, dtype=torch.float32, device=dev)
        self.settings = [torch.zeros(n, dtype=t, device=dev) for t in (torch.float32, torch.int32, torch.float32, torch.float32)]
        self.out = torch.zeros(n, dtype=torch.int64, device=dev)
        self.plan = paged.StepPlan.empty(c.rows, c.page, n, dev, kv_len=c.kv_len, counters=c.counters)
        self.x = torch.zeros(n, dec.cfg.hidden_size, dtype=dec.act, device=dev)
        self.q = torch.zeros(n, dec.H, dec.D, dtype=dec.act, device=dev)
        self.o = torch.zeros_like(self.q)
        self.g = torch.zeros(n, dec.w.intermediate_padded, dtype=dec.act, device=dev)
        self.qkv = torch.zeros(n, dec.cfg.qkv_size, dtype=torch.float32, device=dev)
        self.logits = None
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.graph_launches = 0

    def body(self, planned=lambda: None) -> None:
        """The step; `planned` is called once the plan is launched."""
        d, w, cfg, c = self.d, self.d.w, self.d.cfg, self.d.cache
        eps = cfg.rms_norm_eps
        few = self.n <= GEMV_ROWS
        plan = c.plan(self.add, self.n, out=self.plan)
        planned()
        x = self.x
        x.copy_(K.embedding(self.tokens, w.embed, status=d._word(0)))
        for li, lw in enumerate(w.layers):
            if few:
                qkv = K.gemv(x, lw.wqkv, "f32", bias=lw.bqkv, y_f32=self.qkv, norm_w=lw.in_norm, eps=eps)
            else:
                qkv = K.gemm(K.rmsnorm(x, lw.in_norm, eps), lw.wqkv, "bias" if lw.bqkv is not None else "store", bias=lw.bqkv)
            paged.rope_append_kv8(qkv, d.cos, d.sin, plan.pos, plan.unit, c.block_table, *c.layer(li), heads=d.H,
                                  q_out=self.q, status=d._word(0))
            paged.attention_kv8(self.q, *c.layer(li), c.block_table, c.kv_len, plan.cu, max_q=1, scale=d.scale, out=self.o,
                                want_lse=False, status=d._word(0))
            o = self.o.view(self.n, -1)
            if few:
                K.gemv(o, lw.wo, "residual", y_bf16=x)
                K.gemv(x, lw.wgu, "swiglu", y_bf16=self.g, norm_w=lw.post_norm, eps=eps)
                K.gemv(self.g, lw.wd, "residual", y_bf16=x)
            else:
                x = K.gemm(o, lw.wo, "residual", residual=x)
                g = K.gemm(K.rmsnorm(x, lw.post_norm, eps), lw.wgu, "swiglu")
                x = K.gemm(g, lw.wd, "residual", residual=x)
        self.logits = d._logits(x)
        sampling.sample(self.logits, self.u, *self.settings, out=self.out)

    def run(self, active: int, add, state, tokens, u, *settings) -> torch.Tensor:
        """The step of `add`; `state`: the cache's host mirror after it, taken over with the plan."""
        commit = lambda: self.d.cache.commit(state)  # noqa: E731
        # (from pinned memory, so the host does not wait here for the step before)
        self.add.copy_(torch.tensor(add, dtype=torch.int32, pin_memory=self.d.cuda), non_blocking=True)
        self.tokens[:active].copy_(tokens.reshape(-1))
        for buf, value in zip(self.settings, settings):
            if isinstance(value, torch.Tensor):
                buf[:active].copy_(value.reshape(-1))
            else:
                buf.fill_(value)
        if u is not None:
            self.u[:active].copy_(u.reshape(-1))
        if not self.d.use_graphs:
            self.body(commit)
        else:
            if self.graph is None:
                # nothing runs during the capture: the first replay is the first step
                graph = torch.cuda.CUDAGraph()
                # a garbage collection inside the capture may destroy another graph, which CUDA answers by
                # invalidating the capture
                collects = gc.isenabled()
                gc.disable()
                try:
                    with launches.capture() as cap:
                        with torch.cuda.graph(graph):
                            self.body()
                finally:
                    if collects:
                        gc.enable()
                self.graph, self.graph_launches = graph, cap.launches
            self.graph.replay()
            commit()
            launches.count(self.graph_launches)
        self.d._logits_now = self.logits[:active]
        return self.out[:active].clone()     # (the next step of this size writes `out` again)
