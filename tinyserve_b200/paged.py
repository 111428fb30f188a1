"""Serving over one pool of cache pages: chunked prompts and single tokens in
the same step, sampled continuations.

The reference pages its cache for several requests
(tinyserve/paged_kv_cache.py:20-122) and runs them one at a time
(tinyserve/server.py:48-150).  Here every step is one ragged batch: the next
token of each decoding request together with chunks of the prompts that are
still being read.  Per layer the batch takes the fused q|k|v projection,
``ops.paged_kv_store`` (RoPE, keys and values into their pages),
``ops.paged_attention`` (causal, sliding window and sink logits as the model
has them) and the expert layer; the rows that end a prompt or a decoded token
go through the LM head to ``ops.sample_tokens``.
"""
from __future__ import annotations

import itertools
import operator
from dataclasses import dataclass, field

import torch
import torch.nn.functional as F

from . import ops
from .gptoss import GptOssDecoder
from .moe import ONE_BY_ONE


class PagePool:
    """``pages`` pages of ``page_size`` positions for every layer's keys and
    values, [layers, pages, kv_heads, page_size, head_dim], and the list of the
    free ones.  A page is handed out for all layers at once."""

    def __init__(self, layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype,
                 device: torch.device):
        self.k = torch.zeros(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.page_size = page_size
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free(self) -> int:
        return len(self._free)

    def pages_for(self, positions: int) -> int:
        return -(-positions // self.page_size)

    def take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise RuntimeError(f"{n} pages wanted, {len(self._free)} free")
        return [self._free.pop() for _ in range(n)]

    def give_back(self, pages: list[int]) -> None:
        self._free.extend(reversed(pages))


@dataclass
class PagedRequest:
    request_id: int
    prompt: list[int]
    max_new_tokens: int
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    generated: list[int] = field(default_factory=list)
    logprobs: list[float] = field(default_factory=list)
    logits: list[torch.Tensor] = field(default_factory=list)  # per emitted token, when kept
    pages: list[int] = field(default_factory=list)
    held: int = 0  # positions in the cache
    error: str | None = None  # why the request ended early

    @property
    def done(self) -> bool:
        return len(self.generated) >= self.max_new_tokens


class PagedServingEngine:
    """Continuous batching of a GPT-OSS model whose MoE blocks are QuantMoE
    layers, over a pool of ``pages`` pages.

    chunk_tokens  most new tokens of a step: the decoding requests' first, prompt chunks in what is left
    max_batch     most requests under way at once; a request waits until the pool has pages for its whole length
    seed          of the random numbers behind the sampled tokens
    """

    def __init__(self, model, moe_layers, pages: int = 1024, page_size: int = 64, max_batch: int = 64,
                 max_seq: int = 4096, kv_dtype: torch.dtype = torch.float8_e4m3fn, chunk_tokens: int = 1024,
                 eos_token_id: int | None = None, keep_logits: bool = False, seed: int = 0):
        if chunk_tokens < max_batch:
            raise ValueError("chunk_tokens must cover one token of each of max_batch requests")
        self.dec = d = GptOssDecoder(model, moe_layers, max_seq=1, kv_dtype=kv_dtype)
        rot = model.model.rotary_emb
        p = torch.arange(max_seq, device=d.device, dtype=torch.float32)
        freqs = p[:, None] * rot.inv_freq.float().to(d.device)[None, :]
        self.cos = (freqs.cos() * rot.attention_scaling).to(torch.bfloat16)
        self.sin = (freqs.sin() * rot.attention_scaling).to(torch.bfloat16)
        self.max_batch, self.max_seq, self.chunk_tokens = max_batch, max_seq, chunk_tokens
        self.pool = PagePool(d.L, pages, d.nkv, page_size, d.D, kv_dtype, d.device)
        # the expert layers' scratch for a step of any size; they run one after the other and share it
        need = {False: 0, True: 0}  # by QuantMoE.dense
        for lay in d.layers:
            moe = lay["moe"]
            need[moe.dense] = max([need[moe.dense]] + [moe.workspace_bytes(t) for t in range(ONE_BY_ONE + 1, chunk_tokens + 1)])
        self._expert_ws = {k: torch.zeros(n, dtype=torch.uint8, device=d.device) for k, n in need.items()}
        self._ws = ops.paged_workspace(d.device, d.D)
        # every scratch of a step, each with its error word in front
        self._scratch = [self._ws] + [t for t in self._expert_ws.values() if t.numel()]
        self._scratch += [lay["moe"].workspace(1) for lay in d.layers]
        self.eos = eos_token_id
        self.keep_logits = keep_logits
        self._ids = itertools.count()
        self._rng = torch.Generator(device=d.device).manual_seed(seed)
        self.waiting: list[PagedRequest] = []
        self.running: list[PagedRequest] = []
        self.finished: dict[int, PagedRequest] = {}

    def submit(self, prompt: torch.Tensor, max_new_tokens: int, *, temperature: float = 0.0, top_k: int = 0,
               top_p: float = 1.0, min_p: float = 0.0) -> int:
        """Queue a prompt; temperature 0 decodes greedily, the other settings are ``ops.sample_tokens``'s."""
        ids = prompt.reshape(-1).tolist()
        if not ids:
            raise ValueError("empty prompt")
        vocab = self.dec.embed.shape[0]
        if min(ids) < 0 or max(ids) >= vocab:
            raise ValueError(f"prompt ids must be tokens, 0 to {vocab - 1}")
        temperature, top_p, min_p = float(temperature), float(top_p), float(min_p)
        top_k = operator.index(top_k)
        if not -2 ** 31 <= top_k < 2 ** 31:
            raise ValueError("top_k must fit 32 bits")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be positive")
        if len(ids) + max_new_tokens > self.max_seq:
            raise ValueError("prompt + max_new_tokens exceeds max_seq")
        r = PagedRequest(next(self._ids), ids, max_new_tokens, temperature, top_k, top_p, min_p)
        if self.pool.pages_for(len(ids) + max_new_tokens) > self.pool.k.shape[1]:
            raise ValueError("the request needs more pages than the pool has")
        self.waiting.append(r)
        return r.request_id

    def _admit(self) -> None:
        while self.waiting and len(self.running) < self.max_batch:
            r = self.waiting[0]
            need = self.pool.pages_for(len(r.prompt) + r.max_new_tokens)
            if need > self.pool.free:
                return
            self.waiting.pop(0)
            r.pages = self.pool.take(need)
            self.running.append(r)

    def _plan(self) -> list[tuple[PagedRequest, list[int]]]:
        """The step's requests and the tokens each feeds: a token for every
        decoding request, then prompt chunks while the step has room."""
        room = self.chunk_tokens
        batch = []
        for r in self.running:
            if r.held >= len(r.prompt):
                batch.append((r, r.generated[-1:]))
                room -= 1
        for r in self.running:
            if r.held < len(r.prompt) and room > 0:
                ids = r.prompt[r.held:r.held + room]
                batch.append((r, ids))
                room -= len(ids)
        return batch

    @torch.no_grad()
    def _forward(self, batch: list[tuple[PagedRequest, list[int]]]) -> torch.Tensor:
        """Hidden states (final norm applied) of each request's last fed token, [len(batch), H]."""
        d, pool = self.dec, self.pool
        dev = d.device
        ends, table = [0], []
        width = max(len(r.pages) for r, _ in batch)
        for r, ids in batch:
            ends.append(ends[-1] + len(ids))
            table.append(r.pages + [0] * (width - len(r.pages)))
        host = torch.tensor([t for _, ids in batch for t in ids], dtype=torch.int64)
        tokens = host.to(dev)
        cu = torch.tensor(ends, dtype=torch.int32).to(dev)
        kv = torch.tensor([r.held + len(ids) for r, ids in batch], dtype=torch.int32).to(dev)
        pages = torch.tensor(table, dtype=torch.int32).to(dev)
        max_q = max(len(ids) for _, ids in batch)
        x = d.embed.index_select(0, tokens).float()
        h = torch.empty(x.shape, dtype=torch.bfloat16, device=dev)
        d._norm(x, None, d.layers[0]["ln1"], h)
        for li, lay in enumerate(d.layers):
            qkv = F.linear(h, lay["wqkv"], lay["bqkv"])
            q = ops.paged_kv_store(qkv, self.cos, self.sin, pool.k[li], pool.v[li], pages, cu, kv, n_q_heads=d.nq,
                                   workspace=self._ws)
            a = ops.paged_attention(q, pool.k[li], pool.v[li], pages, cu, kv, max_q, scale=d.scale,
                                    window=d.window if d.sliding[li] else 0, sinks=lay["sinks"],
                                    workspace=self._ws)
            d._norm(x, F.linear(a.view(a.shape[0], -1), lay["wo"], lay["bo"]), lay["ln2"], h)
            moe = lay["moe"]
            y, _, _ = moe.decode(h, out_dtype=torch.float32, workspace=self._expert_ws[moe.dense])
            d._norm(x, y, d._next_norm(li), h)
        return h.index_select(0, (cu[1:] - 1).long())

    def step(self) -> int:
        """Admit waiting requests, run one ragged batch, sample the tokens that
        are due; returns how many requests emitted one."""
        self._admit()
        batch = self._plan()
        if not batch:
            return 0
        last = self._forward(batch)
        for r, ids in batch:
            r.held += len(ids)
        due = [i for i, (r, _) in enumerate(batch) if r.held >= len(r.prompt)]
        emitted = self._emit([batch[i][0] for i in due], last[due] if len(due) < len(batch) else last) if due else 0
        for r in [r for r in self.running if r.done]:
            self.running.remove(r)
            self.pool.give_back(r.pages)
            r.pages = []
            self.finished[r.request_id] = r
        return emitted

    def _device_error(self) -> int:
        """The first error a kernel has reported since the last call, 0 for none; what it left behind is cleared."""
        codes = torch.cat([t[:4].view(torch.int32) for t in self._scratch]).tolist()
        code = next((c for c in codes if c), 0)
        if code:
            for t in self._scratch:
                t.zero_()
        return code

    @torch.no_grad()
    def _emit(self, requests: list[PagedRequest], last: torch.Tensor) -> int:
        logits = F.linear(last, self.dec.lm_head)
        noise = settings = None
        if any(r.temperature > 0 for r in requests):
            noise = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
            noise.exponential_(generator=self._rng)
            dev = logits.device
            settings = dict(temperature=torch.tensor([r.temperature for r in requests], device=dev),
                            top_k=torch.tensor([r.top_k for r in requests], dtype=torch.int32, device=dev),
                            top_p=torch.tensor([r.top_p for r in requests], device=dev),
                            min_p=torch.tensor([r.min_p for r in requests], device=dev))
        tokens, logprobs = ops.sample_tokens(logits, noise, **(settings or {}))
        code = self._device_error()
        if code:
            # of this step or one before that emitted nothing: no cache under way is to be trusted
            for r in self.running:
                r.error = f"device error {code}"
                r.max_new_tokens = len(r.generated)
            return 0
        emitted = 0
        for i, (r, t, lp) in enumerate(zip(requests, tokens.tolist(), logprobs.tolist())):
            if t < 0:
                # nothing to draw from, and nothing to feed: the others of the batch go on without it
                r.error = "no token: every logit is NaN or -infinity"
                r.max_new_tokens = len(r.generated)
                continue
            emitted += 1
            r.generated.append(t)
            r.logprobs.append(lp)
            if self.keep_logits:
                r.logits.append(logits[i].float().cpu())
            if self.eos is not None and t == self.eos:
                r.max_new_tokens = len(r.generated)
        return emitted

    def run(self) -> dict[int, list[int]]:
        """Serve until every submitted request has finished; returns
        {request id: generated token ids}.  A request that could not go on
        ends with what it has; ``finished[id].error`` says why."""
        while self.waiting or self.running:
            self.step()
        return {i: r.generated for i, r in sorted(self.finished.items())}
