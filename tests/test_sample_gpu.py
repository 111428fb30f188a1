"""Token sampling against its definition in 64 bits: equal tokens wherever the
race is decided by more than the rounding of its scores, log-probabilities to
fp32 rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")
    from tinyserve_b200 import ops
    return ops


def settings(rows, vocab, seed):
    rng = np.random.RandomState(seed)
    t = rng.choice([0.0, 0.5, 0.8, 1.0, 2.0], rows)
    k = rng.choice([0, 1, 2, 5, 40, vocab, vocab + 3, -1], rows)
    p = rng.choice([0.0, 0.3, 0.9, 0.99, 1.0, 1.5], rows)
    m = rng.choice([0.0, 0.01, 0.2, 1.0], rows)
    return t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32)


def both(ops, logits, noise, t, k, p, m):
    dev = [None if a is None else torch.as_tensor(a).cuda() for a in (t, k, p, m)]
    tok, lp = ops.sample_tokens(logits, noise, temperature=dev[0], top_k=dev[1], top_p=dev[2], min_p=dev[3])
    rows = logits.shape[0]
    one = [np.ones(rows) if t is None else t, np.zeros(rows, int) if k is None else k,
           np.ones(rows) if p is None else p, np.zeros(rows) if m is None else m]
    want = R.sample(logits.double().cpu().numpy(), noise.double().cpu().numpy(), *[np.asarray(a, float if i != 1 else int)
                                                                                  for i, a in enumerate(one)])
    return tok.cpu().numpy(), lp.double().cpu().numpy(), want


def check(got, logprobs, want, scale=64.0):
    tokens, lp, margins = want
    # scores are fp32 values up to `scale` in size: a handful of roundings of 2^-24 of that
    sure = margins > 8 * scale * 2.0 ** -24
    assert (got[sure] == tokens[sure]).all()
    assert sure.mean() > 0.9
    same = got == tokens
    fin = np.isfinite(lp) & same
    assert (np.abs(logprobs[fin] - lp[fin]) <= 2.0 ** -20 * (1 + np.abs(lp[fin]))).all()
    assert (logprobs[~np.isfinite(lp)] == lp[~np.isfinite(lp)]).all()


def inputs(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype)
    return x, torch.empty(rows, vocab, device="cuda").exponential_(generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (40, 33), (64, 511), (33, 4097), (5, 50001), (2, 201088)])
def test_mixed_settings(ops, rows, vocab, dtype):
    x, e = inputs(rows, vocab, dtype, rows + vocab)
    s = settings(rows, vocab, vocab)
    check(*both(ops, x, e, *s))


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.5, 30.0])
def test_flat_and_peaked_rows(ops, spread):
    """Equal logits (ranked by index alone), nearly equal ones, and rows whose
    mass sits on one token."""
    x, e = inputs(48, 3001, torch.float32, 3, spread)
    check(*both(ops, x, e, *settings(48, 3001, 5)), scale=256.0)


def test_many_ties_at_the_cut(ops):
    """A few distinct logits: the cuts of top-k and top-p fall among equals."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(0, 4, (64, 1000), generator=g, device="cuda").to(torch.bfloat16)
    e = torch.empty(64, 1000, device="cuda").exponential_(generator=g)
    rng = np.random.RandomState(0)
    k = rng.randint(1, 1000, 64).astype(np.int32)
    check(*both(ops, x, e, None, k, None, None))
    # top-p alone: sums of equal weights in 64 bits are exact enough to name the last token
    p = rng.uniform(0.05, 0.95, 64).astype(np.float32)
    check(*both(ops, x, e, None, None, p, None))
    # zeros of either sign are equal
    z = torch.zeros(4, 100, device="cuda")
    z[:, ::2] = -0.0
    check(*both(ops, z, e[:4, :100].contiguous(), None, np.array([1, 3, 50, 99], np.int32), None, None))


@pytest.mark.parametrize("low", [-float("inf"), float("nan"), torch.finfo(torch.float32).min])
def test_masked_logits(ops, low):
    """Tokens ruled out with -inf, NaN or the type's lowest value are not drawn
    while others are left; a row of nothing else gives -1."""
    x, e = inputs(32, 700, torch.float32, 8)
    g = torch.Generator(device="cuda").manual_seed(2)
    hide = torch.rand(32, 700, generator=g, device="cuda") < 0.9
    hide[3] = True
    hide[4] = True
    hide[4, 123] = False
    x[hide] = low
    got, lp, want = both(ops, x, e, *settings(32, 700, 6))
    check(got, lp, want, scale=256.0)
    ruled = hide.cpu().numpy()
    if low == torch.finfo(torch.float32).min:
        assert 0 <= got[3] < 700
    else:
        assert got[3] == -1 and lp[3] == -np.inf
    assert got[4] == 123
    rest = [i for i in range(32) if i != 3]
    assert not ruled[rest, got[rest]].any()


def test_infinite_logits_and_noise_at_its_ends(ops):
    x, e = inputs(16, 300, torch.float32, 9)
    x[:8, 77] = float("inf")
    x[:4, 200] = float("inf")
    e[8:, 50] = 0.0
    e[8:, 51] = float("inf")
    got, lp, want = both(ops, x, e, None, None, None, None)
    assert (got == want[0]).all()
    assert set(got[:4]) <= {77, 200} and (got[4:8] == 77).all() and (got[8:] == 50).all()


def test_extreme_temperatures(ops):
    x, e = inputs(6, 500, torch.float32, 10)
    x[:, 3] = -float("inf")
    t = np.array([1e-30, 1e-45, 1e30, np.inf, np.nan, -2.0], np.float32)
    tok, lp = ops.sample_tokens(x, e, temperature=torch.tensor(t).cuda())
    best = x.argmax(1)
    assert tok[0] == best[0] and tok[1] == best[1] and tok[4] == best[4] and tok[5] == best[5]
    flat = e.clone()
    flat[:, 3] = float("inf")
    assert tok[2] == flat[2].argmin() and tok[3] == flat[3].argmin()
    assert not torch.isnan(lp).any()


def test_strides_defaults_and_greedy(ops):
    x, e = inputs(20, 1000, torch.float16, 11)
    wide_x = torch.zeros(20, 1111, dtype=torch.float16, device="cuda")
    wide_e = torch.ones(20, 1001, device="cuda")
    wide_x[:, 3:1003], wide_e[:, 1:] = x, e  # rows that start anywhere
    a = ops.sample_tokens(x, e)
    b = ops.sample_tokens(wide_x[:, 3:1003], wide_e[:, 1:])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(*both(ops, x, e, None, None, None, None))
    tok, lp = ops.sample_tokens(x)
    first = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, 0]
    assert torch.equal(tok, first)
    ref = torch.log_softmax(x.double(), 1).gather(1, first[:, None])[:, 0]
    assert ((lp - ref).abs() <= 2.0 ** -20 * (1 + ref.abs())).all()
    t = torch.zeros(20, device="cuda")
    assert torch.equal(ops.sample_tokens(x, e, temperature=t)[0], first)
    again = [ops.sample_tokens(x, e, top_p=torch.full((20,), 0.7, device="cuda")) for _ in range(3)]
    assert all(torch.equal(again[0][i], r[i]) for r in again for i in (0, 1))


def test_distribution(ops):
    """20,000 rows of one distribution: chi-square of the drawn counts against
    the kept, renormalised probabilities (5 degrees of freedom; the statistic
    exceeds 40 with probability 1.5e-7)."""
    logits = torch.tensor([2.0, 1.5, 1.0, 0.5, 0.0, -0.5, -6.0, -7.0], device="cuda").repeat(20000, 1)
    g = torch.Generator(device="cuda").manual_seed(12)
    e = torch.empty(20000, 8, device="cuda").exponential_(generator=g)
    tok, _ = ops.sample_tokens(logits, e, top_k=torch.full((20000,), 6, dtype=torch.int32, device="cuda"))
    count = torch.bincount(tok, minlength=8).double().cpu()
    want = torch.softmax(logits[0, :6].double(), 0).cpu() * 20000
    assert count[6:].sum() == 0
    assert float(((count[:6] - want) ** 2 / want).sum()) < 40


def test_refusals(ops):
    x, e = inputs(4, 10, torch.float32, 0)
    for error, f in (
            (RuntimeError, lambda: ops.sample_tokens(x.cpu(), e)), (ValueError, lambda: ops.sample_tokens(x.double(), e)),
            (ValueError, lambda: ops.sample_tokens(x[0], e[0])), (ValueError, lambda: ops.sample_tokens(x, e[:2])),
            (ValueError, lambda: ops.sample_tokens(x, e.half())), (ValueError, lambda: ops.sample_tokens(x[:, :0])),
            (ValueError, lambda: ops.sample_tokens(x.t().contiguous().t(), e)),
            (RuntimeError, lambda: ops.sample_tokens(x[:1].expand(4, 10), e)),
            (ValueError, lambda: ops.sample_tokens(x, e, temperature=torch.ones(3, device="cuda"))),
            (ValueError, lambda: ops.sample_tokens(x, e, top_k=torch.ones(4, device="cuda"))),
            (ValueError, lambda: ops.sample_tokens(x, e, top_p=torch.ones(4, device="cuda").double()))):
        with pytest.raises(error):
            f()
    tok, lp = ops.sample_tokens(x[:0], e[:0])
    assert tok.shape == lp.shape == (0,)


@pytest.mark.parametrize("likely", [6000, 9000])
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_likely_tokens_side_by_side(ops, rows, likely):
    """What top-p (or a large k) keeps lies in neighbouring tokens, so that few
    warps of a cluster's CTAs hold all of it: their first lists overflow and
    the bin of the limit is collected alone."""
    x, e = inputs(rows, 201088, torch.float32, rows + likely, spread=0.3)
    x[:, 70000:70000 + likely] += 12.0
    p = np.linspace(0.5, 0.95, rows).astype(np.float32)
    check(*both(ops, x, e, None, None, p, None))
    k = np.full(rows, 2000, np.int32)
    check(*both(ops, x, e, None, k, p, None))


@pytest.mark.parametrize("best,level", [(100, 30000), (5000, 1000), (3000, 3000)])
def test_top_p_that_ends_with_a_level(ops, best, level):
    """Three levels of equal logits, top-p within a few roundings of the mass of
    the first two: no more than the first token or so of the last level is
    kept, and none of the better ones is lost."""
    rows, vocab = 160, 60000  # one CTA a row
    x = torch.full((rows, vocab), -30.0, device="cuda")
    e = torch.ones(rows, vocab, device="cuda")
    a = torch.linspace(0.3, 3.0, rows, dtype=torch.float64).float().cuda()
    x[:, :best] = 0.0
    x[:, best:best + level] = -a[:, None]
    tail = slice(best + level, best + level + 2000)
    x[:, tail] = -2.0 * a[:, None]
    w = torch.exp(x.double())
    limit = (w[:, :best + level].sum(1) / w.sum(1)).cpu().numpy()
    e[:, best + level + 1000] = 1e-12  # in the middle of the last level: would win if kept
    e[:, 7] = 1e-6                     # of the best level: wins
    for ulps in range(-3, 4):
        p = limit.astype(np.float32)
        for _ in range(abs(ulps)):
            p = np.nextafter(p, np.float32(2.0 if ulps > 0 else 0.0))
        tok, _ = ops.sample_tokens(x, e, top_p=torch.from_numpy(p).cuda())
        assert (tok == 7).all(), (ulps, tok[tok != 7][:5])
