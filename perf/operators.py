"""Serving operators around a paged KV cache, measured case by case.

Three operators that one serving step runs one after the other:

* ``store``: rotate the new tokens' queries and keys (RoPE) and put keys and values into their pages.
* ``attention``: attend from a ragged batch of new tokens (prompt chunks and single decode tokens together) over the
  paged cache; causal, optionally a sliding window with a few first tokens that stay visible, optionally a sink
  logit per head in the softmax denominator.
* ``sample``: draw the next token of each row from its logits with temperature, top-k, top-p and min-p, by an
  exponential race over given random numbers, with the log-probability of the drawn token.

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, through the package's
entry points.  ``exact`` is the same from the definitions in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases
def _attention(name, seqs, new, context, heads, page, dtype, cache, window=0, keep_first=0, sinks=True, ragged=True,
               mix=1):
    return {"name": name, "op": "attention", "seqs": seqs, "new": new, "context": context, "q_heads": heads[0],
            "kv_heads": heads[1], "head_dim": heads[2], "page": page, "dtype": dtype, "cache": cache,
            "window": window, "keep_first": keep_first, "sinks": sinks, "ragged": ragged, "mix": mix}


def _store(name, seqs, new, context, heads, page, dtype, cache, tables, ragged=True, mix=1):
    return {"name": name, "op": "store", "seqs": seqs, "new": new, "context": context, "q_heads": heads[0],
            "kv_heads": heads[1], "head_dim": heads[2], "page": page, "dtype": dtype, "cache": cache,
            "tables": tables, "ragged": ragged, "mix": mix}


def _sample(name, rows, vocab, dtype, filters, mix=1):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters, "mix": mix}


def listed():
    gpt_oss = (64, 8, 64)  # the whole-model decoder's heads: 64 query heads in 8 groups of 64 dimensions
    return [
        # the 64 rows of a full serving step: one new token each
        _store("store_step_64", 64, 1, 64, gpt_oss, 16, "bf16", "same", "bf16"),
        # a long prompt admitted in one go, into an 8-bit cache
        _store("store_prompt_8192_e4m3", 1, 8192, 8192, gpt_oss, 64, "bf16", "e4m3", "f32", ragged=False),
        # the smallest call: one request's single token, a short context; latency is all
        _attention("decode_1x500", 1, 1, 500, gpt_oss, 16, "bf16", "same", ragged=False),
        # a full serving step over 64 ragged contexts with the 8-bit cache, a full-attention layer
        _attention("decode_64x4096_e4m3", 64, 1, 4096, gpt_oss, 64, "bf16", "e4m3"),
        # the same batch in a sliding layer that keeps the first tokens visible, 16-bit cache
        _attention("decode_64x8191_window", 64, 1, 8191, gpt_oss, 16, "bf16", "same", window=128, keep_first=4),
        # a whole prompt at once: the largest product
        _attention("prompt_4096", 1, 4096, 4096, gpt_oss, 64, "bf16", "same", ragged=False),
        # a later chunk of a long prompt over what the 8-bit cache holds already
        _attention("chunk_1024_of_8192_e4m3", 1, 1024, 8192, gpt_oss, 64, "bf16", "e4m3", ragged=False),
        # chunks and single tokens together, wide heads, windowed, odd sizes, no sink logit, one idle slot
        _attention("mixed_9x500_wide", 9, 500, 2047, (32, 8, 128), 24, "f16", "same", window=1000, keep_first=5,
                   sinks=False),
        # one request's token at the model's vocabulary
        _sample("sample_1x201088", 1, 201088, "f32", "top_p"),
        # a full serving step, every row with its own settings
        _sample("sample_64x201088", 64, 201088, "bf16", "mixed"),
        # no filter: the whole row races
        _sample("sample_32x201088_plain", 32, 201088, "f32", "none"),
        # many rows, a small odd vocabulary
        _sample("sample_200x32001", 200, 32001, "f16", "top_k"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    mix = rng.randrange(1 << 20)
    heads = rng.choice([(64, 8, 64), (32, 8, 128), (16, 16, 64), (24, 2, 64), (40, 8, 128), (14, 2, 64), (8, 1, 128)])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice(["same", "e4m3"])
    what = rng.choice(["store", "decode", "decode", "chunk", "chunk", "mixed", "sample", "sample"])
    if what == "store":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 8192 // seqs)
        case = _store("", seqs, new, new + rng.randrange(0, 65), heads, page, dtype, cache,
                      rng.choice(["bf16", "f32"]), rng.random() < 0.7, mix)
    elif what == "sample":
        vocab = _log(rng, 500, 201088)
        case = _sample("", _log(rng, 1, min(256, 64 * 201088 // vocab)), vocab, rng.choice(["f32", "bf16", "f16"]),
                       rng.choice(["none", "top_k", "top_p", "min_p", "mixed"]), mix)
    else:
        # never more than the listed cases hold: the whole prompt's products, 64 x 4096 cached positions in a step
        most = 4096 * 4096 * 4096 // (2 * heads[0] * heads[2])
        if what == "decode":
            seqs, new = _log(rng, 1, 64), rng.choice([1, 1, 1, 2])
            context = _log(rng, 16, 64 * 4096 // seqs if seqs > 8 else 32768)
        elif what == "chunk":
            seqs, new = 1, _log(rng, 3, int(most ** 0.5))
            context = _log(rng, new, min(32768, most // new))
        else:
            seqs, new = _log(rng, 2, 16), _log(rng, 8, 1024)
            context = _log(rng, new, max(new, min(8192, most // (new * seqs))))
        window = 0 if rng.random() < 0.5 else _log(rng, 8, context + 1)
        case = _attention("", seqs, new, context, heads, page, dtype, cache, window,
                          rng.choice([0, 1, 4, 19]) if window else 0, rng.random() < 0.7, rng.random() < 0.7, mix)
    del case["name"]
    return case


def _lengths(case):
    """New tokens and cached positions (the new ones included) of each sequence: fixed by the case."""
    rng = random.Random(case["mix"])
    n, new, context = case["seqs"], case["new"], case["context"]
    if not case["ragged"]:
        return [new] * n, [context] * n
    q = [new if i == 0 else 1 if rng.random() < 0.4 else _log(rng, 1, new) for i in range(n)]
    kv = [context if i == n // 2 and q[i] <= context else rng.randint(max(q[i], context // 8), context)
          for i in range(n)]
    if n >= 4 and new > 1:
        q[-1], kv[-1] = 0, 0  # an idle slot of the batch
    return q, kv


def _settings(case):
    """Temperature, top-k, top-p and min-p of each row: fixed by the case."""
    rng = random.Random(case["mix"])
    t, k, p, m = [], [], [], []
    for i in range(case["rows"]):
        kind = case["filters"] if case["filters"] != "mixed" else ("none", "top_k", "top_p", "min_p", "all", "greedy")[i % 6]
        t.append(0.0 if kind == "greedy" else rng.choice([0.6, 0.7, 1.0, 1.3]))
        k.append(min(case["vocab"], _log(rng, 5, 200)) if kind in ("top_k", "all") else 0)
        p.append(rng.choice([0.8, 0.9, 0.95]) if kind in ("top_p", "all") else 1.0)
        m.append(rng.choice([0.02, 0.05, 0.1]) if kind in ("min_p", "all") else 0.0)
    return t, k, p, m


# ---------------------------------------------------------------------------------------------------------- inputs
def _cuda_rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _batch(case, rng):
    """Lengths and page table of a ragged batch: pages in a shuffled order, a few of the pool unused."""
    q, kv = _lengths(case)
    page = case["page"]
    used = [-(-n // page) for n in kv]
    width = max(1, max(used))
    pool = sum(used) + 3
    order = torch.randperm(pool, generator=rng, device="cuda").to(torch.int32)
    table = torch.zeros(len(q), width, dtype=torch.int64)
    take = 0
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(take, take + n)
        take += n
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    return {"page_table": order[table.cuda()], "cu_q": torch.tensor(cu, dtype=torch.int32, device="cuda"),
            "kv_lens": torch.tensor(kv, dtype=torch.int32, device="cuda"), "max_q": max(q), "tokens": cu[-1],
            "pool": pool}


def prepare(case, seed):
    rng = _cuda_rng(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn(rows, vocab, generator=rng, device="cuda") * 2.5
        # a few likely continuations stand out, as a trained model's do
        best = torch.randint(vocab, (rows, 8), generator=rng, device="cuda")
        logits.scatter_add_(1, best, torch.rand(rows, 8, generator=rng, device="cuda") * 9)
        noise = torch.empty(rows, vocab, device="cuda").exponential_(generator=rng)
        t, k, p, m = _settings(case)
        return {"op": "sample", "logits": logits.to(_TYPES[case["dtype"]]), "noise": noise,
                "temperature": torch.tensor(t, device="cuda"),
                "top_k": torch.tensor(k, dtype=torch.int32, device="cuda"),
                "top_p": torch.tensor(p, device="cuda"), "min_p": torch.tensor(m, device="cuda")}
    s = _batch(case, rng)
    nq, nkv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = _TYPES[case["dtype"]]
    held = torch.float8_e4m3fn if case["cache"] == "e4m3" else dtype
    s |= {"op": case["op"], "q_heads": nq}
    if case["op"] == "store":
        s["qkv"] = torch.randn(s["tokens"], (nq + 2 * nkv) * d, generator=rng, device="cuda").to(dtype)
        angle = (torch.arange(case["context"], device="cuda", dtype=torch.float32)[:, None]
                 * 150000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
        s["cos"], s["sin"] = angle.cos().to(_TYPES[case["tables"]]), angle.sin().to(_TYPES[case["tables"]])
        s["k_cache"] = torch.zeros(s["pool"], nkv, page, d, device="cuda", dtype=held)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        return s
    s["q"] = torch.randn(s["tokens"], nq, d, generator=rng, device="cuda").to(dtype)
    shape = (s["pool"], nkv, page, d)
    s["k_cache"] = (torch.randn(shape, generator=rng, device="cuda") * 1.5).to(held)
    s["v_cache"] = torch.randn(shape, generator=rng, device="cuda").to(held)
    s["sinks"] = torch.randn(nq, generator=rng, device="cuda") if case["sinks"] else None
    s["window"], s["keep_first"], s["scale"] = case["window"], case["keep_first"], d ** -0.5
    return s


# ---------------------------------------------------------------------------------------------------------- passes
def run(s):
    if own:
        from tinyserve_b200 import ops
        if s["op"] == "store":
            q = ops.paged_kv_store(s["qkv"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["page_table"],
                                   s["cu_q"], s["kv_lens"], n_q_heads=s["q_heads"])
            return {"q": q, "k": _values(s["k_cache"]), "v": _values(s["v_cache"])}
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["cu_q"], s["kv_lens"],
                                       s["max_q"], scale=s["scale"], window=s["window"],
                                       keep_first=s["keep_first"], sinks=s["sinks"])
        tokens, logprobs = ops.sample_tokens(s["logits"], s["noise"], temperature=s["temperature"],
                                             top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    return {"store": _plain_store, "attention": _plain_attention, "sample": _plain_sample}[s["op"]](s)


def _values(cache):
    """What an 8-bit cache stands for; a wider one as it is."""
    return cache.to(torch.bfloat16) if cache.element_size() == 1 else cache


def _places(s, n):
    """Sequence, index in it and position of each of the batch's n new tokens."""
    token = torch.arange(n, device="cuda")
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    seq = torch.searchsorted(cu[1:], token, right=True)
    at = token - cu[seq]
    return seq, at, kv[seq] - (cu[seq + 1] - cu[seq]) + at


def _plain_store(s):
    qkv, kc, vc = s["qkv"], s["k_cache"], s["v_cache"]
    n, (_, nkv, page, d), nq = qkv.shape[0], kc.shape, s["q_heads"]
    seq, _, pos = _places(s, n)
    x = qkv.float().view(n, nq + 2 * nkv, d)
    turned, v = x[:, :nq + nkv], x[:, nq + nkv:]
    cos, sin = s["cos"].float()[pos][:, None], s["sin"].float()[pos][:, None]
    a, b = turned[..., :d // 2], turned[..., d // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(qkv.dtype)
    place, row = s["page_table"].long()[seq, pos // page], pos % page
    kc[place, :, row] = turned[:, nq:].to(kc.dtype)
    vc[place, :, row] = v.to(qkv.dtype).to(vc.dtype)
    return {"q": turned[:, :nq].contiguous(), "k": _values(kc), "v": _values(vc)}


def _plain_attention(s):
    q, table = s["q"], s["page_table"].long()
    n, nq, d = q.shape
    _, nkv, page, _ = s["k_cache"].shape
    seqs, most, group = table.shape[0], s["max_q"], nq // nkv
    keys = s["k_cache"][table].float().permute(0, 2, 1, 3, 4).reshape(seqs, nkv, -1, d)
    values = s["v_cache"][table].float().permute(0, 2, 1, 3, 4).reshape(seqs, nkv, -1, d)
    seq, at, pos = _places(s, n)
    padded = torch.zeros(seqs, most, nq, d, device="cuda")
    padded[seq, at] = q.float()
    padded = padded.view(seqs, most, nkv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, nkv, group * most, d)
    scores = torch.matmul(padded, keys.transpose(2, 3)).mul_(s["scale"]).view(seqs, nkv, group, most, -1)
    j = torch.arange(scores.shape[-1], device="cuda")
    where = torch.full((seqs, most), -1, device="cuda", dtype=torch.long)
    where[seq, at] = pos
    where = where[..., None]
    seen = j <= where
    if s["window"]:
        seen &= (j > where - s["window"]) | (j < s["keep_first"])
    scores = scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, nkv, group, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    weight = scores.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(weight.view(seqs, nkv, group * most, -1), values).view(seqs, nkv, group, most, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, most, nq, d)[seq, at].to(q.dtype)


def _plain_sample(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    top, greedy = x.amax(1, keepdim=True), (s["temperature"] <= 0)[:, None]
    inverse = torch.where(greedy, torch.ones_like(top), 1.0 / s["temperature"][:, None])
    scaled = (x - top) * inverse
    weight = torch.exp(scaled)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices  # equal logits: the lower index first
    ranked = weight.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(s["top_k"] <= 0, vocab, s["top_k"])[:, None]
    ranked = torch.where(rank < k, ranked, torch.zeros_like(ranked))
    before = torch.cumsum(ranked, 1) - ranked
    p = s["top_p"][:, None]
    kept = (rank < k) & ((before < p * ranked.sum(1, keepdim=True)) | (p >= 1)) & (ranked >= s["min_p"][:, None])
    kept[:, 0] = True
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    race = torch.where(greedy, x, scaled - torch.log(s["noise"])).masked_fill_(~kept, float("-inf"))
    best = race.amax(1, keepdim=True)
    tokens = torch.where(race == best, rank, vocab).amin(1)
    logprobs = scaled.gather(1, tokens[:, None])[:, 0] - torch.log(weight.sum(1))
    return {"tokens": tokens, "logprobs": logprobs}


# ---------------------------------------------------------------------------------------------------------- floors
def work(case):
    if case["op"] == "sample":
        rows, vocab, size = case["rows"], case["vocab"], _TYPES[case["dtype"]].itemsize
        t, k, p, m = _settings(case)
        # a row without a filter reads its random numbers too, and a filtered one only those of what it keeps
        whole = sum(1 for i in range(rows) if t[i] > 0 and k[i] == 0 and p[i] >= 1 and m[i] <= 0)
        return {"bytes": rows * vocab * size + 4 * whole * vocab + 28 * rows, "flops": 4 * rows * vocab}
    q, kv = _lengths(case)
    nq, nkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    size, held = 2, 1 if case["cache"] == "e4m3" else 2
    n = sum(q)
    tables = 4 * sum(-(-x // case["page"]) for x in kv) + 8 * len(q)
    if case["op"] == "store":
        trig = (4 if case["tables"] == "f32" else 2) * d * n
        return {"bytes": n * d * ((nq + 2 * nkv) * size + nq * size + 2 * nkv * held) + trig + tables,
                "flops": 3 * n * (nq + nkv) * d}
    pairs = positions = 0
    w, f = case["window"], case["keep_first"]
    for a, b in zip(q, kv):
        if not a:
            continue
        p = np.arange(b - a, b, dtype=np.int64)
        low = np.maximum(0, p - w + 1) if w else np.zeros_like(p)
        pairs += int((p + 1 - low + np.minimum(low, f)).sum())
        first = int(low[0])
        positions += b - first + min(first, f)
    return {"bytes": 2 * n * nq * d * size + 2 * positions * nkv * d * held + tables, "flops": 4 * d * nq * pairs}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    q_lens, kv_lens = _lengths(case)
    if case["op"] == "store":
        return _exact_store(case, s, q_lens, kv_lens)
    return _exact_attention(case, s, q_lens, kv_lens)


def _rows_of(case, s, b, length):
    """Pool rows (page, place in it) of a sequence's first `length` positions."""
    j = torch.arange(length, device="cuda")
    return s["page_table"][b].long()[j // case["page"]], j % case["page"]


def _exact_store(case, s, q_lens, kv_lens):
    nq, nkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    k, v = s["k_cache"].double(), s["v_cache"].double()
    out, at = [], 0
    for b, (new, length) in enumerate(zip(q_lens, kv_lens)):
        rows = s["qkv"][at:at + new].double().view(new, nq + 2 * nkv, d)
        at += new
        c, z = (s[t][length - new:length].double()[:, None] for t in ("cos", "sin"))
        lo, hi = rows[:, :nq + nkv, :d // 2], rows[:, :nq + nkv, d // 2:]
        both = torch.empty_like(rows[:, :nq + nkv])
        both[..., :d // 2] = lo * c - hi * z
        both[..., d // 2:] = lo * z + hi * c
        out.append(both[:, :nq])
        page, place = (t[length - new:] for t in _rows_of(case, s, b, length))
        k[page, :, place] = both[:, nq:]
        v[page, :, place] = rows[:, nq + nkv:]
    return {"q": torch.cat(out), "k": k, "v": v}


def _exact_attention(case, s, q_lens, kv_lens):
    nq, nkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    group, out, at = nq // nkv, [], 0
    for b, (new, length) in enumerate(zip(q_lens, kv_lens)):
        if not new:
            continue
        page, place = _rows_of(case, s, b, length)
        j = torch.arange(length, device="cuda")
        p = torch.arange(length - new, length, device="cuda")[:, None]
        hidden = j > p
        if case["window"]:
            hidden |= (p - j >= case["window"]) & (j >= case["keep_first"])
        rows = torch.empty(new, nq, d, device="cuda", dtype=torch.float64)
        for h in range(nkv):
            keys, values = (s[t][page, h, place].double() for t in ("k_cache", "v_cache"))
            for g in range(h * group, (h + 1) * group):
                logit = s["q"][at:at + new, g].double() @ keys.T / math.sqrt(d)
                logit[hidden] = -math.inf
                if s["sinks"] is not None:
                    logit = torch.cat([logit, s["sinks"][g].double().expand(new, 1)], 1)
                rows[:, g] = torch.softmax(logit, 1)[:, :length] @ values
        out.append(rows)
        at += new
    return torch.cat(out)


def _exact_sample(s):
    tokens, logprobs = [], []
    x, noise = s["logits"].double().cpu().numpy(), s["noise"].double().cpu().numpy()
    t, k, p, m = (s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p"))
    for i in range(x.shape[0]):
        row = x[i] / (t[i] if t[i] > 0 else 1.0)
        mass = np.exp(row - row.max())
        ranked = np.argsort(-x[i], kind="stable")
        if k[i] > 0:
            ranked = ranked[:int(k[i])]
        if p[i] < 1:
            cum = np.cumsum(mass[ranked])
            ranked = ranked[:1 + int(np.searchsorted(cum[:-1], p[i] * cum[-1], side="left"))]
        ranked = ranked[(mass[ranked] >= m[i]) | (np.arange(len(ranked)) == 0)]
        if t[i] > 0:
            ranked = np.sort(ranked)
            best = int(ranked[np.argmin(noise[i][ranked] / mass[ranked])])
        else:
            best = int(ranked[0])
        tokens.append(best)
        logprobs.append(row[best] - row.max() - math.log(mass.sum()))
    return {"tokens": torch.tensor(tokens), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
