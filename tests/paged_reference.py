"""The paged operators from their definitions in 64 bits, for the tests: no
code of the package, and none of the tolerances."""
from __future__ import annotations

import math

import numpy as np
import torch


class Batch:
    """A ragged batch with its pools: sequence b has q_lens[b] new tokens, the
    last of its kv_lens[b] positions.  Pages are handed out in a shuffled
    order, ``spare`` of the pool stay unused; everything no position lives
    in (unused pages, page tails) is filled with ``fill``."""

    def __init__(self, q_lens, kv_lens, nq, nkv, d, page, dtype, held, seed=0, spare=3, fill=float("nan"),
                 layout="heads", device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.page = list(q_lens), list(kv_lens), page
        self.nq, self.nkv, self.d, self.dtype, self.held = nq, nkv, d, dtype, held
        used = [-(-n // page) for n in self.kv_lens]
        pool, width = sum(used) + spare, max(used + [0]) + 1
        order = torch.randperm(pool, generator=g).to(torch.int32)
        table = torch.full((len(used), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table
        shape = (pool, nkv, page, d)
        self.k = torch.full(shape, fill)
        self.v = torch.full(shape, fill)
        for b, n in enumerate(self.kv_lens):
            j = torch.arange(n)
            pg, row = table[b, j // page].long(), j % page
            self.k[pg, :, row] = torch.randn(n, nkv, d, generator=g) * 1.3
            self.v[pg, :, row] = torch.randn(n, nkv, d, generator=g)
        self.k, self.v = self.k.to(held), self.v.to(held)
        if layout == "rows":  # stored [pages, rows, heads, D], passed as [pages, heads, rows, D]
            self.k, self.v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (self.k, self.v))
        self.n = sum(self.q_lens)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(self.q_lens)]), dtype=torch.int32)
        self.kv = torch.tensor(self.kv_lens, dtype=torch.int32)
        self.q = torch.randn(self.n, nq, d, generator=g).to(dtype)
        self.sinks = torch.randn(nq, generator=g)
        self.max_q = max(self.q_lens + [0])
        if device:
            self.to(device)

    def to(self, device):
        keep = {}
        for name in ("table", "k", "v", "cu", "kv", "q", "sinks"):
            t = getattr(self, name)
            moved = t.to(device)
            if t.stride() != moved.stride():
                moved = t.transpose(1, 2).contiguous().to(device).transpose(1, 2)
            keep[name] = moved
        self.__dict__.update(keep)
        return self

    def cached(self, pool, b, h):
        """The values sequence b holds in KV head h, float64 [kv_len, D]."""
        j = np.arange(self.kv_lens[b])
        table = self.table[b].cpu().numpy()
        idx = torch.tensor(table[j // self.page], dtype=torch.long, device=pool.device)
        row = torch.tensor(j % self.page, dtype=torch.long, device=pool.device)
        return pool.float()[idx, h, row].double().cpu().numpy() if len(j) else np.zeros((0, self.d))


def attention(batch, scale=None, window=0, keep_first=0, sinks=True):
    """(out, magnitude) float64 [N, nq, D]: the attention and sum_j w_j |v_j|,
    the size that the roundings of weights and sums are relative to."""
    scale = batch.d ** -0.5 if scale is None else scale
    q = batch.q.double().cpu().numpy()
    s0 = batch.sinks.double().cpu().numpy()
    out, mag = np.zeros_like(q), np.zeros_like(q)
    at = 0
    for b, (n, length) in enumerate(zip(batch.q_lens, batch.kv_lens)):
        for h in range(batch.nkv):
            k, v = batch.cached(batch.k, b, h), batch.cached(batch.v, b, h)
            for g in range(batch.nq // batch.nkv):
                head = h * (batch.nq // batch.nkv) + g
                for i in range(n):
                    p = length - n + i
                    see = np.arange(max(0, p + 1))
                    if window:
                        see = see[(see > p - window) | (see < keep_first)]
                    if not len(see):
                        continue
                    s = scale * (k[see] @ q[at + i, head])
                    m = max(s.max(), s0[head]) if sinks else s.max()
                    w = np.exp(s - m)
                    w /= w.sum() + (math.exp(s0[head] - m) if sinks else 0.0)
                    out[at + i, head] = w @ v[see]
                    mag[at + i, head] = w @ np.abs(v[see])
        at += n
    return out, mag


def sample(logits, noise, temperature, top_k, top_p, min_p):
    """(tokens, logprobs, race margins) of float64 rows; the margin is the gap
    between the two best of the race (infinite for one candidate)."""
    tokens, logprobs, margins = [], [], []
    for x, e, t, k, p, m in zip(logits, noise, temperature, top_k, top_p, min_p):
        x = np.where(np.isnan(x), -np.inf, x)
        top = x.max()
        if top == -np.inf:
            tokens.append(-1), logprobs.append(-np.inf), margins.append(np.inf)
            continue
        with np.errstate(invalid="ignore"):
            d = np.where(x == top, 0.0, (x - top) / (t if t > 0 else 1.0)) if top < np.inf else \
                np.where(x == np.inf, 0.0, -np.inf)
        w = np.exp(d)
        order = np.argsort(-x, kind="stable")
        kept = order[:k] if k > 0 else order
        if p < 1:
            before = np.cumsum(w[kept]) - w[kept]
            kept = kept[before < p * w[kept].sum()] if p > 0 else kept[:1]
        kept = np.concatenate([kept[:1], kept[1:][(w[kept[1:]] >= m) & (w[kept[1:]] > 0)]]) if len(kept) else order[:1]
        if t > 0:
            with np.errstate(divide="ignore"):
                race = d[kept] - np.log(e[kept])
            best = race.max()
            token = int(kept[race == best].min())
            rest = race[kept != token]
            margin = best - rest.max() if len(rest) else np.inf
        else:
            token, margin = int(order[0]), np.inf
        tokens.append(token), margins.append(margin)
        logprobs.append(d[token] - np.log(w.sum()))
    return np.array(tokens), np.array(logprobs), np.array(margins)
