"""The paged serving engine's bookkeeping around a stand-in for the model (no GPU)."""
from __future__ import annotations

import itertools
from types import SimpleNamespace

import pytest
import torch

from tinyserve_b200 import paged

VOCAB, HIDDEN = 32, 8


@pytest.fixture
def engine(monkeypatch):
    """An engine whose forward pass gives zeros and whose sampler gives the
    tokens of ``script`` (a list per call), recording what is fed."""
    eng = paged.PagedServingEngine.__new__(paged.PagedServingEngine)
    eng.dec = SimpleNamespace(lm_head=torch.zeros(VOCAB, HIDDEN, dtype=torch.bfloat16), device=torch.device("cpu"),
                              embed=torch.zeros(VOCAB, HIDDEN, dtype=torch.bfloat16), layers=[])
    eng.max_batch, eng.max_seq, eng.chunk_tokens = 4, 64, 16
    eng.pool = paged.PagePool(1, 20, 1, 4, 64, torch.bfloat16, torch.device("cpu"))
    eng.eos, eng.keep_logits = None, False
    eng._ids, eng._rng = itertools.count(), torch.Generator()
    eng.waiting, eng.running, eng.finished = [], [], {}
    eng._scratch = [torch.zeros(64, dtype=torch.uint8) for _ in range(2)]
    eng.fed, eng.script = [], []

    def forward(batch):
        eng.fed.append([list(ids) for _, ids in batch])
        assert all(0 <= t < VOCAB for _, ids in batch for t in ids)
        return torch.zeros(len(batch), HIDDEN, dtype=torch.bfloat16)

    def sample(logits, noise=None, **kw):
        tokens = eng.script.pop(0) if eng.script else [1] * logits.shape[0]
        assert len(tokens) == logits.shape[0]
        return torch.tensor(tokens), torch.zeros(len(tokens))

    eng._forward = forward
    monkeypatch.setattr(paged.ops, "sample_tokens", sample)
    return eng


def test_a_request_without_a_token_ends_alone(engine):
    """sample_tokens gives -1 for a row of no finite logit: that request ends
    with an error and gives its pages back; the others go on."""
    ids = [engine.submit(torch.tensor([3, 4, 5]), 4) for _ in range(3)]
    engine.script = [[7, 8, 9], [10, -1, 11]]
    out = engine.run()
    assert out == {ids[0]: [7, 10, 1, 1], ids[1]: [8], ids[2]: [9, 11, 1, 1]}
    assert engine.finished[ids[1]].error and engine.pool.free == 20
    assert engine.finished[ids[0]].error is None and engine.finished[ids[2]].error is None
    engine.script = [[-1]]
    first = engine.submit(torch.tensor([3]), 2)
    assert engine.run()[first] == [] and engine.finished[first].error


def test_submit_refuses_what_a_step_could_not_take(engine):
    """Ids that are no token would index past the embedding, a top_k past 32
    bits would fail the whole batch's step."""
    for bad in (dict(prompt=torch.tensor([3, VOCAB])), dict(prompt=torch.tensor([-1])), dict(top_k=2 ** 31),
                dict(top_k=-2 ** 31 - 1), dict(top_k=1.5), dict(temperature="warm"), dict(top_p=None)):
        a = dict(prompt=torch.tensor([3, 4]), max_new_tokens=2) | bad
        with pytest.raises((ValueError, TypeError)):
            engine.submit(a.pop("prompt"), a.pop("max_new_tokens"), **a)
    assert not engine.waiting
    rid = engine.submit(torch.tensor([0, VOCAB - 1]), 2, temperature=1, top_k=2 ** 31 - 1, top_p=0.5, min_p=0)
    assert engine.run()[rid] == [1, 1]


def test_device_errors_end_what_is_under_way(engine):
    """An error word that a kernel set: no token of that step is handed out, the
    requests under way end with an error, those that wait are served after."""
    ids = [engine.submit(torch.tensor([3, 4, 5]), 3) for _ in range(5)]  # one more than max_batch
    engine.step()
    engine._scratch[1].fill_(1)
    assert engine.step() == 0
    for i in ids[:4]:
        assert engine.finished[i].generated == [1] and "device error" in engine.finished[i].error
    assert engine.pool.free == 20 and not any(t.any() for t in engine._scratch)
    assert engine.run()[ids[4]] == [1, 1, 1] and engine.finished[ids[4]].error is None
