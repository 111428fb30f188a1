"""Serving over pages (tinyserve_b200.paged.PagedServingEngine) against the
batch-1 decoder on the same small GPT-OSS model: chunked prompts and single
tokens in one batch, pages given back and taken again, sampled tokens."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")
    from transformers import GptOssConfig

    from tinyserve_b200.offload import load_and_offload
    cfg = GptOssConfig(hidden_size=512, intermediate_size=256, num_hidden_layers=2, num_local_experts=8,
                       num_experts_per_tok=2, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
                       vocab_size=512, sliding_window=4, layer_types=["sliding_attention", "full_attention"])
    return load_and_offload(cfg, device="cuda", seed=21)


def prompts(lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=g) for n in lens]


def engine(lm, **kw):
    from tinyserve_b200.paged import PagedServingEngine
    a = dict(pages=40, page_size=16, max_batch=8, max_seq=128, chunk_tokens=32, keep_logits=True) | kw
    return PagedServingEngine(lm.model, lm.moe_layers, **a)


class Routing:
    """Records what the expert layers are given and choose while it is on."""

    def __init__(self, lm):
        self.lm, self.calls = lm, []

    def __enter__(self):
        for li, layer in enumerate(self.lm.moe_layers):
            def record(x, *args, _decode=layer.decode, _li=li, **kw):
                out = _decode(x, *args, **kw)
                self.calls.append((_li, x.detach().clone(), out[1].detach().clone()))
                return out
            layer.decode = record
        return self

    def __exit__(self, *_):
        for layer in self.lm.moe_layers:
            del layer.decode


def serve_recorded(lm, eng):
    """Runs the engine; {request id: {position: per layer the chosen experts}}."""
    chosen = {}
    forward = eng._forward

    def recorded(batch):
        with Routing(lm) as log:
            out = forward(batch)
        at = 0
        for r, ids in batch:
            for n in range(len(ids)):
                chosen.setdefault(r.request_id, {})[r.held + n] = [set(c[2][at + n].tolist()) for c in log.calls]
            at += len(ids)
        return out

    eng._forward = recorded
    eng.run()
    return chosen


def check_against_decoder(lm, req, kv_dtype, chosen):
    """Logits within the bound that the slot-based engine's tests hold (bf16
    projections as a batch against single rows), as long as both routed alike.
    Where they did not, the two experts' logits have to lie within 2% of the
    largest (hidden states differ by half a percent, and bf16 logits tie); from
    there on the two caches hold different values.  Returns the number of
    tokens compared."""
    from tinyserve_b200.gptoss import GptOssDecoder
    whole = req.prompt + req.generated[:-1]
    dec = GptOssDecoder(lm.model, lm.moe_layers, max_seq=128, kv_dtype=kv_dtype, prefill_chunk=128)
    with Routing(lm) as log:
        dec.prefill(torch.tensor(whole).cuda())
    alike = len(whole)
    for li, x, ids in log.calls:
        layer = lm.moe_layers[li]
        logits = x.float() @ layer.router_w.float().T
        if layer.router_b is not None:
            logits = logits + layer.router_b.float()
        ranked = logits.sort(dim=1, descending=True).values
        k = ids.shape[1]
        for pos in range(len(whole)):
            if chosen[pos][li] != set(ids[pos].tolist()) and pos < alike:
                assert float(ranked[pos, k - 1] - ranked[pos, k]) < 0.02 * float(ranked[pos].abs().max())
                alike = pos
    dec = GptOssDecoder(lm.model, lm.moe_layers, max_seq=128, kv_dtype=kv_dtype, prefill_chunk=4)
    compared = 0
    for i in range(len(req.generated)):
        got = dec.prefill(torch.tensor(req.prompt).cuda()) if i == 0 else dec.step(req.generated[i - 1])
        got = got if i == 0 else dec._logits[0].float()
        if len(req.prompt) + i <= alike:
            assert rel_l2(req.logits[i].numpy(), got.cpu().numpy()) < 1e-2
            compared += 1
    return compared


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("page_size,chunk", [(16, 32), (5, 9)])
def test_matches_the_single_request_decoder(lm, kv, page_size, chunk):
    """More requests than fit, prompts longer than a step, decoding beside prompts."""
    lens, news = (5, 50, 3, 21, 1, 9), (6, 4, 7, 3, 5, 8)
    eng = engine(lm, kv_dtype=kv, page_size=page_size, chunk_tokens=chunk, pages=160 // page_size, max_batch=4)
    ids = [eng.submit(p, m) for p, m in zip(prompts(lens), news)]
    chosen = serve_recorded(lm, eng)
    assert sorted(eng.finished) == ids and [len(eng.finished[i].generated) for i in ids] == list(news)
    assert eng.pool.free == 160 // page_size
    compared = 0
    for i in ids:
        req = eng.finished[i]
        compared += check_against_decoder(lm, req, kv, chosen[i])
        assert req.generated == [int(x.argmax()) for x in req.logits]
    assert compared >= sum(news) // 2
    from tinyserve_b200 import ops
    assert ops.paged_device_error() == 0


def test_sampled_requests(lm):
    """top_k = 1 is greedy whatever the temperature; a seed repeats its tokens;
    log-probabilities are those of the logits at the request's temperature."""
    def serve(seed, **kw):
        eng = engine(lm, seed=seed)
        ids = [eng.submit(p, 6, **kw) for p in prompts((5, 20, 3))]
        eng.run()
        return [eng.finished[i] for i in ids]

    greedy = [r.generated for r in serve(0)]
    assert [r.generated for r in serve(1, temperature=1.5, top_k=1)] == greedy
    assert [r.generated for r in serve(2, temperature=0.7, min_p=1.0)] == greedy
    a, b, c = (serve(s, temperature=1.2, top_k=40, top_p=0.95) for s in (7, 7, 8))
    assert [r.generated for r in a] == [r.generated for r in b] != [r.generated for r in c]
    for r in a:
        for x, t, lp in zip(r.logits, r.generated, r.logprobs):
            want = torch.log_softmax(x.double() / 1.2, -1)[t]
            assert abs(float(want) - lp) < 1e-5 * (1 + abs(lp))
            assert int((x > x[t]).sum()) < 40


def test_eos_and_refusals(lm):
    eng = engine(lm)
    first = eng.submit(prompts((7,))[0], 9)
    token = eng.run()[first][0]
    eng = engine(lm, eos_token_id=token)
    rid = eng.submit(prompts((7,))[0], 9)
    assert eng.run()[rid] == [token] and eng.pool.free == 40
    for bad in (lambda: eng.submit(torch.zeros(0, dtype=torch.long), 3), lambda: eng.submit(prompts((7,))[0], 0),
                lambda: eng.submit(prompts((120,))[0], 9), lambda: engine(lm, chunk_tokens=4),
                lambda: engine(lm, pages=2).submit(prompts((40,))[0], 9)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="pages"):
        eng.pool.take(41)


def test_steps_of_any_size_take_no_more_memory(lm):
    """Steps of 40 to 17 tokens, then of 16 to 1, after one of the largest: the
    scratch of the expert layers does not grow with the sizes met."""
    eng = engine(lm, chunk_tokens=40, keep_logits=False)

    def serve(n):
        eng.submit(prompts((n,))[0], 1)
        eng.run()
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated()

    serve(40)
    few = serve(16)
    assert all(serve(n) <= few + (1 << 20) for n in [*range(39, 16, -1), *range(15, 0, -1)])


def test_device_errors_are_read(lm):
    """A page that is none in a request's list: the requests of that step end with an error, later ones are served."""
    eng = engine(lm)
    first = eng.submit(prompts((20,))[0], 4)
    eng.step()
    eng.running[0].pages[0] = 10 ** 6
    eng.step()
    assert "device error" in eng.finished[first].error and len(eng.finished[first].generated) == 1
    eng.pool._free = list(range(40))
    again = eng.submit(prompts((20,))[0], 4)
    eng.run()
    assert eng.finished[again].error is None and len(eng.finished[again].generated) == 4
