"""Paged KV store and paged attention against their definitions in 64 bits, at
the lengths, masks, page sizes and layouts where they can go wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu

BF, F16, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
# half an ulp of the 16-bit types, relative: bf16 has 8 significant bits, f16 has 11
HALF_ULP = {BF: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("CUDA required")
    from tinyserve_b200 import ops
    return ops


def attend(ops, b, **kw):
    sinks = b.sinks if kw.pop("sinks", True) else None
    return ops.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, b.max_q, sinks=sinks, **kw)


def check(got, b, **kw):
    """Weights and the output are each rounded once to a 16-bit type (half an
    ulp u of |out| and of the magnitude sum w |v|); scores are fp32 sums of up
    to 128 products of size below 32 (error below 2^-13 each, so 2^-12 of the
    magnitude after exp, and the sums of weights); f16 also has its smallest
    step."""
    ref, mag = R.attention(b, **kw)
    u = HALF_ULP[b.dtype]
    got = got.double().cpu().numpy()
    bound = u * np.abs(ref) + (u + 2.0 ** -12) * mag + 2.0 ** -24
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - ref) / bound) if got.size else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the bound"


# new tokens and cached positions: single tokens, a first prompt, chunks that end inside a page or a tile,
# an idle slot, more new tokens than positions (rows that see nothing)
RAGGED = ([1, 1, 0, 7, 33, 1, 5, 130], [1, 300, 0, 7, 100, 129, 3, 150])
SINGLE = ([1] * 6, [1, 2, 64, 65, 511, 1000])
SHORT = ([2, 3, 1, 2], [2, 40, 17, 260])
PROMPT = ([257, 1, 16], [257, 16, 16])


@pytest.mark.parametrize("held", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d,heads", [(64, (8, 1)), (64, (4, 4)), (128, (6, 2)), (128, (16, 1)), (64, (14, 2))])
@pytest.mark.parametrize("lens", [RAGGED, SINGLE, SHORT, PROMPT], ids=["ragged", "single", "short", "prompt"])
def test_attention(ops, lens, d, heads, dtype, held):
    b = R.Batch(*lens, *heads, d, 16, dtype, E4 if held == "e4m3" else dtype, seed=d + heads[0])
    check(attend(ops, b), b)


@pytest.mark.parametrize("page", [1, 8, 24, 100, 256])
@pytest.mark.parametrize("lens", [RAGGED, SINGLE], ids=["ragged", "single"])
def test_page_sizes(ops, page, lens):
    b = R.Batch(*lens, 8, 2, 64, page, BF, BF, seed=page)
    check(attend(ops, b), b)


@pytest.mark.parametrize("held", [BF, E4])
@pytest.mark.parametrize("sinks", [True, False])
@pytest.mark.parametrize("window,keep", [(1, 0), (1, 3), (37, 0), (37, 4), (128, 1), (128, 140), (5000, 4)])
def test_window_and_first_tokens(ops, window, keep, sinks, held):
    for lens in (RAGGED, ([1, 1, 3, 1], [900, 129, 500, 20]), ([200], [640])):
        b = R.Batch(*lens, 8, 2, 64, 16, BF, held, seed=window + keep)
        kw = dict(window=window, keep_first=keep, sinks=sinks)
        check(attend(ops, b, **kw), b, **kw)


def test_long_contexts_are_split(ops):
    """Few rows over many positions: the key range is divided and joined."""
    for lens in (([1], [20011]), ([3, 1], [9000, 12345]), ([40], [6001])):
        b = R.Batch(*lens, 8, 1, 64, 64, BF, E4, seed=5)
        check(attend(ops, b), b)


def test_rows_that_see_nothing_are_zero(ops):
    b = R.Batch([4, 20], [0, 2], 8, 2, 64, 16, BF, BF)
    for sinks in (True, False):
        out = attend(ops, b, sinks=sinks)
        assert (out[:4] == 0).all() and (out[4:22] == 0).all() and (out[22:] != 0).any()
        check(out, b, sinks=sinks)


@pytest.mark.parametrize("held", [BF, E4])
@pytest.mark.parametrize("q,kv", [(40, 300), (2, 70), (1, 90)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_the_mask_hides_does_not_matter(ops, bad, q, kv, held):
    """NaN and infinities in keys and values that a row may not see: later
    tokens of its chunk, positions before its window, page tails and unused
    pages (filled with NaN by the batch).  The rows that do see them are NaN or
    infinite, and only those."""
    if held == E4 and bad == float("inf"):
        bad = float("nan")  # e4m3 has no infinity
    b = R.Batch([q], [kv], 8, 2, 64, 16, BF, held, seed=q)
    window, keep = 30, 2
    clean = attend(ops, b, window=window, keep_first=keep)
    check(clean, b, window=window, keep_first=keep)
    late, early = kv - 1 - q // 2, max(keep, kv - q - window)  # seen by the later rows; by no row
    for pool in (b.k, b.v):
        for j in {early} | ({late + 1} if q > 1 else set()):
            page, row = int(b.table[0, j // 16]), j % 16
            pool[page, :, row] = torch.tensor(bad).to(held)
    out = attend(ops, b, window=window, keep_first=keep)
    p = torch.arange(kv - q, kv, device="cuda")
    hit = torch.zeros(q, dtype=torch.bool, device="cuda")
    for j in {early} | ({late + 1} if q > 1 else set()):
        hit |= (j <= p) & ((j > p - window) | (j < keep))
    assert torch.equal(out[~hit], clean[~hit])
    assert not torch.isfinite(out[hit]).any()


def test_values_alone_hidden_by_the_mask(ops):
    """Only a value is not finite: its row of V meets a weight of zero."""
    for q, kv in ((50, 50), (200, 333), (2, 40)):
        b = R.Batch([q], [kv], 8, 1, 64, 16, BF, BF, seed=kv)
        clean = attend(ops, b)
        j = kv - 1
        b.v[int(b.table[0, j // 16]), :, j % 16, 5] = float("inf")
        out = attend(ops, b)
        assert torch.equal(out[:-1], clean[:-1])
        assert torch.equal(out[-1, :, :5], clean[-1, :, :5]) and torch.equal(out[-1, :, 6:], clean[-1, :, 6:])
        assert (out[-1, :, 5] == float("inf")).all()


@pytest.mark.parametrize("held", [BF, E4])
def test_layouts_and_strides(ops, held):
    """Pools stored by rows, q as a view of the fused projection, padding rows."""
    for lens in (RAGGED, SINGLE):
        b = R.Batch(*lens, 8, 2, 64, 16, BF, held, layout="rows")
        assert not b.k.is_contiguous()
        qkv = torch.randn(b.n + 5, 12, 64, device="cuda").to(BF)
        qkv[:b.n, :8] = b.q
        out = torch.full((b.n + 5, 8, 64), 7.0, dtype=BF, device="cuda")
        ops.paged_attention(qkv[:, :8], b.k, b.v, b.table, b.cu, b.kv, b.max_q, sinks=b.sinks, out=out)
        check(out[:b.n], b)
        assert (out[b.n:] == 7.0).all()  # rows of no sequence


def test_large_scores_and_scales(ops):
    """One key far above the rest at either end, a negative and a zero scale."""
    for lens in (([1, 3], [400, 300]), ([150], [400])):
        b = R.Batch(*lens, 8, 1, 64, 16, BF, BF, seed=9)
        for j in (0, 255, 299):
            b.k[int(b.table[0, j // 16]), :, j % 16] *= 16
        for scale in (1.0, -0.125, 0.0):
            ref, mag = R.attention(b, scale=scale)
            got = attend(ops, b, scale=scale).double().cpu().numpy()
            # scores reach 16 * 64 * 20 * scale: fp32 sums of 64 products err by 2^-18 of that size
            err = 2.0 ** -12 + 2 * 64 * 20 * 20 * abs(scale) * 2.0 ** -18
            assert (np.abs(got - ref) <= HALF_ULP[BF] * np.abs(ref) + (HALF_ULP[BF] + err) * mag + 1e-30).all()


def test_wide_range_of_q(ops):
    """q of either end of bf16's range over an 8-bit cache, and tiny ones."""
    for size in (1e-30, 1e-6, 3e4, 1e30):
        for lens in (([1], [100]), ([40], [100])):
            b = R.Batch(*lens, 8, 1, 64, 16, BF, E4, seed=3)
            b.q = (b.q.float() * size).to(BF)
            check(attend(ops, b, scale=0.125 / size), b, scale=0.125 / size)


def test_offsets_beyond_32_bits(ops):
    """Pages that start past 2^32 elements of the pool."""
    b = R.Batch([1, 40], [100, 60], 8, 1, 64, 16, BF, E4, seed=1)
    far = (1 << 32) // 1024 + 7
    for name in ("k", "v"):
        small = getattr(b, name)
        big = torch.empty(far + small.shape[0], 1, 16, 64, dtype=E4, device="cuda")
        big[far:] = small
        setattr(b, name, big)
    b.table[b.table >= 0] += far
    out = attend(ops, b)
    b.k, b.v, b.table = b.k[far:], b.v[far:], torch.where(b.table >= 0, b.table - far, b.table)
    check(out, b)


def test_same_result_every_time_and_on_another_stream(ops):
    for lens in (([1, 1], [5000, 77]), RAGGED):
        b = R.Batch(*lens, 8, 2, 64, 16, BF, BF)
        first = attend(ops, b)
        for _ in range(3):
            assert torch.equal(attend(ops, b), first)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            out = attend(ops, b)
        st.synchronize()
        assert torch.equal(out, first)


def test_in_a_graph(ops):
    """Captured once, replayed with other lengths and tables in place."""
    b = R.Batch([1, 1, 20], [300, 900, 50], 8, 2, 64, 16, BF, BF, seed=1)
    other = R.Batch([1, 1, 20], [800, 5, 200], 8, 2, 64, 16, BF, BF, seed=2, spare=0)
    pool = max(b.k.shape[0], other.k.shape[0])
    for t in (b, other):
        for n in ("k", "v"):
            grown = torch.zeros(pool, 2, 16, 64, dtype=BF, device="cuda")
            grown[:getattr(t, n).shape[0]] = getattr(t, n)
            setattr(t, n, grown)
        table = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
        table[:, :t.table.shape[1]] = t.table
        t.table = table
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        attend(ops, b)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = attend(ops, b)
        g.replay()
        st.synchronize()
        check(out, b)
        for n in ("k", "v", "q", "kv", "table", "sinks"):
            getattr(b, n).copy_(getattr(other, n))
        g.replay()
        st.synchronize()
    check(out, other)


@pytest.mark.parametrize("held", ["same", "e4m3"])
@pytest.mark.parametrize("tables", ["same", "f32", "other"])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_store(ops, d, dtype, tables, held):
    """Rotated q and k within one rounding of the 64-bit product (and three of
    fp32), what is stored exactly that rounded value (e4m3: rounded once
    more), nothing else of the pools touched."""
    nq, nkv = 6, 2
    b = R.Batch(RAGGED[0], [max(q, k) for q, k in zip(*RAGGED)], nq, nkv, d, 24, dtype, E4 if held == "e4m3" else dtype,
                fill=0.25)
    g = torch.Generator().manual_seed(d)
    wide = torch.randn(b.n, (nq + 2 * nkv) * d + 16, generator=g).to(dtype).cuda()
    qkv = wide[:, :(nq + 2 * nkv) * d]
    ang = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)[None, :]
    other = F16 if dtype == BF else BF
    held_in = {"f32": torch.float32, "same": dtype, "other": other}[tables]
    cos, sin = (t.to(held_in).cuda() for t in (ang.cos(), ang.sin()))
    k0, v0 = b.k.clone(), b.v.clone()
    q = ops.paged_kv_store(qkv, cos, sin, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=nq)
    x = qkv.double().view(b.n, nq + 2 * nkv, d)
    pos = torch.cat([torch.arange(k - n, k) for n, k in zip(b.q_lens, b.kv_lens)]).cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(b.q_lens)]).cuda()
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    ref = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    size = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
    u = HALF_ULP[dtype]

    def near(got, want, m):
        assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -22 * m + 2.0 ** -25).all()

    near(q, ref[:, :nq], size[:, :nq])
    cf, sf, lf, hf = c.float(), s.float(), lo.float()[:, :nq], hi.float()[:, :nq]
    assert torch.equal(q, torch.cat([lf * cf - hf * sf, hf * cf + lf * sf], -1).to(dtype))  # one rounding each
    page, row = b.table[seq, pos // 24].long(), pos % 24
    if held == "same":
        near(b.k[page, :, row], ref[:, nq:nq + nkv], size[:, nq:nq + nkv])
        assert torch.equal(b.v[page, :, row], qkv.reshape(b.n, nq + 2 * nkv, d)[:, nq + nkv:])
    else:
        # the 16-bit value a 16-bit cache gets, rounded once more
        k16, v16 = torch.zeros_like(b.k, dtype=dtype), torch.zeros_like(b.v, dtype=dtype)
        ops.paged_kv_store(qkv, cos, sin, k16, v16, b.table, b.cu, b.kv, n_q_heads=nq)
        for pool, pool16 in ((b.k, k16), (b.v, v16)):
            assert torch.equal(pool.view(torch.uint8)[page, :, row], pool16[page, :, row].to(E4).view(torch.uint8))
    untouched = torch.ones(b.k.shape[0], 24, dtype=torch.bool, device="cuda")
    untouched[page, row] = False
    for pool, before in ((b.k, k0), (b.v, v0)):
        keep = untouched[:, None, :, None].expand_as(pool)
        assert torch.equal(pool.float()[keep], before.float()[keep])


@pytest.mark.parametrize("dtype", [BF, F16])
def test_store_beyond_the_range_of_e4m3(ops, dtype):
    """Values around and past 448, infinities and NaN become what a plain cast makes of them."""
    x = torch.tensor([447.0, 448.0, 456.0, 464.0, 465.0, 466.0, 480.0, 1000.0, 6e4, float("inf"), float("nan"), 0.0,
                      2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10, 2.0 ** -14, 17.3, 0.013])
    x = torch.cat([x, -x, torch.linspace(-470, 470, 28)]).to(dtype).cuda()
    qkv = torch.zeros(1, 3 * 64, dtype=dtype, device="cuda")
    qkv[0, 64:128], qkv[0, 128:] = x, x.flip(0)
    one, zero = torch.ones(1, 32, device="cuda"), torch.zeros(1, 32, device="cuda")
    k = torch.zeros(1, 1, 16, 64, dtype=E4, device="cuda")
    v = torch.zeros_like(k)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cu, kv = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int32).cuda()
    ops.paged_kv_store(qkv, one, zero, k, v, table, cu, kv, n_q_heads=1)
    want = qkv[0].to(E4).float()
    fin = torch.isfinite(x.float())  # x * 1 - y * 0 is NaN next to an infinity, in the other half too
    fin = fin & fin.roll(32)
    assert torch.equal(v[0, 0, 0].float().nan_to_num(nan=-1.0), want[128:].nan_to_num(nan=-1.0))
    assert torch.equal(k[0, 0, 0].float()[fin].nan_to_num(nan=-1.0), want[64:128][fin].nan_to_num(nan=-1.0))
    assert torch.isnan(k[0, 0, 0].float()[~fin]).all()


def test_store_then_attend(ops):
    """A prompt in chunks through both operators equals it in one go."""
    nq, nkv, d, n = 8, 2, 64, 150
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(n, (nq + 2 * nkv) * d, generator=g).to(BF).cuda()
    ang = torch.arange(n)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)[None, :]
    cos, sin = ang.cos().cuda(), ang.sin().cuda()

    def through(cuts):
        k = torch.zeros(12, nkv, 16, d, dtype=BF, device="cuda")
        v = torch.zeros_like(k)
        table = torch.arange(11, -1, -1, dtype=torch.int32, device="cuda")[None]
        outs, at = [], 0
        for c in cuts:
            cu = torch.tensor([0, c], dtype=torch.int32, device="cuda")
            kv = torch.tensor([at + c], dtype=torch.int32, device="cuda")
            q = ops.paged_kv_store(qkv[at:at + c], cos, sin, k, v, table, cu, kv, n_q_heads=nq)
            outs.append(ops.paged_attention(q, k, v, table, cu, kv, c, window=60, keep_first=3))
            at += c
        return torch.cat(outs), k, v

    whole, k1, v1 = through([n])
    parts, k2, v2 = through([64, 1, 1, 33, 51])
    assert torch.equal(k1, k2) and torch.equal(v1, v2)
    # both hold the bound of one rounding of the weights and one of the output
    assert ((whole.float() - parts.float()).abs() <= 4 * HALF_ULP[BF] * (whole.float().abs() + v1.float().abs().max())).all()


def test_inconsistent_batches_are_reported_not_read(ops):
    """A page outside the pool, a length beyond the table, a cu_q that runs past
    the rows or above max_q: device error 2, and the sound sequences are served."""
    good = R.Batch([1, 2, 40], [50, 60, 70], 8, 2, 64, 16, BF, BF)
    want = attend(ops, good)
    assert ops.paged_device_error() == 0
    for what in ("page", "length", "rows", "max_q"):
        b = R.Batch([1, 2, 40], [50, 60, 70], 8, 2, 64, 16, BF, BF)
        if what == "page":
            b.table[2, 1] = b.k.shape[0]
        elif what == "length":
            b.kv[2] = 16 * b.table.shape[1] + 1
        elif what == "rows":
            b.cu[3] += 1
        else:
            b.max_q = 39
        out = attend(ops, b)
        assert torch.equal(out[:3], want[:3]), what
        assert ops.paged_device_error() == 2, what
        assert ops.paged_device_error() == 0
    b = R.Batch([4], [50], 8, 2, 64, 16, BF, BF)
    qkv = torch.zeros(4, 12 * 64, dtype=BF, device="cuda")
    t = torch.zeros(48, 32, device="cuda")  # two positions short
    k0 = b.k.clone()
    b.table[0, 2] = -5
    ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8)
    assert ops.paged_device_error() == 2
    changed = (b.k.view(torch.int16) != k0.view(torch.int16)).any(-1).any(1)  # [page, row]
    assert changed.sum() == 0  # 46 and 47 fall in the missing page, 48 and 49 past the tables


def test_empty_calls(ops):
    b = R.Batch([0, 0], [5, 0], 8, 2, 64, 16, BF, BF)
    assert attend(ops, b).shape == (0, 8, 64)
    b = R.Batch([], [], 8, 2, 64, 16, BF, BF)
    assert attend(ops, b).shape == (0, 8, 64)
    qkv = torch.zeros(0, 12 * 64, dtype=BF, device="cuda")
    t = torch.zeros(4, 32, device="cuda")
    assert ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8).shape == (0, 8, 64)


def test_refusals(ops):
    b = R.Batch([1], [5], 8, 2, 64, 16, BF, BF)

    def call(**kw):
        a = dict(q=b.q, k=b.k, v=b.v, table=b.table, cu=b.cu, kv=b.kv, max_q=1, sinks=b.sinks) | kw
        more = {n: a.pop(n) for n in list(a) if n not in ("q", "k", "v", "table", "cu", "kv", "max_q")}
        return ops.paged_attention(*a.values(), **more)

    for error, kw in (
            (RuntimeError, dict(q=b.q.cpu())), (TypeError, dict(q=b.q.float())), (TypeError, dict(q=b.q.half())),
            (ValueError, dict(q=b.q[0])), (ValueError, dict(q=b.q[..., :32])),
            (ValueError, dict(v=b.v[:, :1])), (ValueError, dict(v=b.v.transpose(1, 2).contiguous().transpose(1, 2))),
            (ValueError, dict(k=b.k.transpose(2, 3), v=b.v.transpose(2, 3))),
            (ValueError, dict(table=b.table.long())), (ValueError, dict(table=b.table[0])),
            (ValueError, dict(cu=b.cu.long())), (ValueError, dict(cu=b.cu[:1])), (ValueError, dict(kv=b.kv.long())),
            (ValueError, dict(sinks=b.sinks.double())), (ValueError, dict(sinks=b.sinks[:4])),
            (ValueError, dict(out=torch.empty(1, 8, 64, device="cuda"))),
            (RuntimeError, dict(window=-1)), (RuntimeError, dict(keep_first=-1)), (RuntimeError, dict(max_q=-1)),
            (RuntimeError, dict(q=b.q.repeat(1, 2, 1)[:, :9], sinks=None)),
            (RuntimeError, dict(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))),
            (RuntimeError, dict(k=b.k[..., :32].contiguous(), v=b.v[..., :32].contiguous(),
                                q=b.q[..., :32].contiguous()))):
        with pytest.raises(error):
            call(**kw)
    odd = torch.zeros(64 * 16 * 2 * 8 + 1, dtype=BF, device="cuda")[1:].view(8, 2, 16, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        call(k=odd, v=odd)
    t = torch.zeros(8, 32, device="cuda")
    qkv = torch.zeros(1, 12 * 64, dtype=BF, device="cuda")
    for kw in (dict(cos=t[:, :16]), dict(cos=t.double(), sin=t.double()), dict(qkv=qkv[:, :64]),
               dict(q_out=torch.empty(1, 8, 64, device="cuda"))):
        a = dict(qkv=qkv, cos=t, sin=t) | kw
        more = {"q_out": a.pop("q_out")} if "q_out" in a else {}
        with pytest.raises(ValueError):
            ops.paged_kv_store(a["qkv"], a["cos"], a["sin"], b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8, **more)


def padded(b, rows):
    """q and out with ``rows`` rows, those past the batch's own of no sequence."""
    q = torch.zeros(rows, b.nq, b.d, dtype=b.dtype, device="cuda")
    q[:b.n] = b.q
    return q, torch.full_like(q, 7.0)


@pytest.mark.parametrize("held", [BF, E4])
@pytest.mark.parametrize("q_lens,most", [([8, 1], 8), ([2], 64), ([32, 1], 32), ([3, 0, 40, 2], 40), ([1, 1, 1], 5)])
def test_buffer_of_full_length_for_every_sequence(ops, q_lens, most, held):
    """As many rows as n_seqs sequences of max_q new tokens need, of which the
    sequences at hand take fewer: every one of theirs is served."""
    b = R.Batch(q_lens, [90 + 7 * i for i in range(len(q_lens))], 8, 1, 64, 16, BF, held, seed=most)
    q, out = padded(b, most * len(q_lens))
    ops.paged_attention(q, b.k, b.v, b.table, b.cu, b.kv, most, sinks=b.sinks, out=out)
    check(out[:b.n], b)
    assert (out[b.n:] == 7.0).all()


def test_graph_of_full_sequences_replayed_with_shorter_ones(ops):
    """Captured with every sequence at its longest, replayed with other cu_q."""
    full = R.Batch([32, 32], [100, 70], 8, 1, 64, 16, BF, BF, seed=1)
    less = R.Batch([31, 2], [95, 66], 8, 1, 64, 16, BF, BF, seed=2)
    pool = max(full.k.shape[0], less.k.shape[0])
    for t in (full, less):
        for n in ("k", "v"):
            grown = torch.zeros(pool, 1, 16, 64, dtype=BF, device="cuda")
            grown[:getattr(t, n).shape[0]] = getattr(t, n)
            setattr(t, n, grown)
        table = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
        table[:, :t.table.shape[1]] = t.table
        t.table = table
    q, out = padded(full, 64)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ops.paged_attention(q, full.k, full.v, full.table, full.cu, full.kv, 32, sinks=full.sinks, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.paged_attention(q, full.k, full.v, full.table, full.cu, full.kv, 32, sinks=full.sinks, out=out)
        g.replay()
        st.synchronize()
        check(out, full)
        for n in ("k", "v", "kv", "table", "sinks", "cu"):
            getattr(full, n).copy_(getattr(less, n))
        q[:less.n] = less.q
        out.fill_(7.0)
        g.replay()
        st.synchronize()
    check(out[:less.n], less)
    assert (out[less.n:] == 7.0).all()


def test_rows_that_overlap_are_refused(ops):
    """qkv rows that share memory (an expanded row, a window sliding over a
    vector) do not hold what the operator would read behind the first."""
    b = R.Batch([3], [5], 8, 2, 64, 16, BF, BF)
    t = torch.rand(8, 32, device="cuda")
    width = 12 * 64
    row = torch.zeros(width + 16, dtype=BF, device="cuda")
    for qkv in (row[:width].expand(3, width), row.as_strided((3, width), (8, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8)
    b = R.Batch([1], [5], 8, 2, 64, 16, BF, BF)
    one = torch.randn(1, width, device="cuda").to(BF)
    want = ops.paged_kv_store(one, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8)
    got = ops.paged_kv_store(one.as_strided((1, width), (0, 1)), t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8)
    assert torch.equal(got, want)  # the stride of a single row says nothing


def captured(f, pool=None):
    """A graph of f() on the capture stream that all such graphs share, without a warm-up there."""
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        out = f()
    return g, out


def test_first_calls_inside_captures(ops):
    """Graphs captured on a stream that has run no paged operator: each holds its
    own scratch, so the second may run before the first, beside it, or
    without it, and calls outside any graph are not touched by either."""
    a = R.Batch([1, 2], [3000, 2000], 8, 1, 64, 16, BF, BF, seed=1)  # both are divided and joined
    b = R.Batch([1, 30], [2500, 2100], 8, 1, 64, 16, BF, BF, seed=2)
    want = [attend(ops, t) for t in (a, b)]
    # memory that is not zero where the graphs take theirs; they run one by one
    g0, junk = captured(lambda: torch.full((64 << 20,), 0x5A, dtype=torch.uint8, device="cuda"))
    del junk
    a_out, b_out = torch.empty_like(a.q), torch.empty_like(b.q)
    ga, _ = captured(lambda: attend(ops, a, out=a_out), g0.pool())
    gb, _ = captured(lambda: attend(ops, b, out=b_out), g0.pool())
    for order in ((gb, ga), (ga, gb)):
        for g in order:
            g0.replay(), g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a_out, want[0]) and torch.equal(b_out, want[1])
    # with memory of their own they may overlap
    ga, out_a = captured(lambda: attend(ops, a))
    gb, out_b = captured(lambda: attend(ops, b))
    for _ in range(2):
        gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_b, want[1])
    ga.replay()
    torch.cuda.synchronize()
    assert torch.equal(out_a, want[0])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        out_a.fill_(7.0), out_b.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            ga.replay()
        with torch.cuda.stream(s2):
            gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_a, want[0]) and torch.equal(out_b, want[1])
    assert torch.equal(attend(ops, a), want[0])
    qkv = torch.randn(31, 10 * 64, device="cuda").to(BF)
    t = torch.rand(2500, 32, device="cuda")
    q = ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8)
    gs, out = captured(lambda: ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8))
    gs.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, q)


def test_errors_inside_captures_are_read(ops):
    """A graph without a workspace of its own reports to the error word that paged_device_error reads."""
    b = R.Batch([1, 2], [50, 60], 8, 1, 64, 16, BF, BF)
    g, _ = captured(lambda: attend(ops, b))
    g.replay()
    assert ops.paged_device_error() == 0
    b.table[1, 1] = b.k.shape[0]
    g.replay()
    assert ops.paged_device_error() == 2
    assert ops.paged_device_error() == 0


@pytest.mark.parametrize("window,keep", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (60, 2 ** 31 - 1), (60, 2 ** 31 - 100),
                                         (511, 3), (512, 3), (2000, 5)])
@pytest.mark.parametrize("held", [BF, E4])
def test_windows_and_first_tokens_of_any_size(ops, window, keep, held):
    """Windows and first tokens up to the integers' end, around the table's
    positions, with rows before the first position."""
    for lens in (RAGGED, ([300, 8], [450, 5]), ([1, 2], [500, 1])):
        b = R.Batch(*lens, 8, 1, 64, 16, BF, held, seed=7)
        kw = dict(window=window, keep_first=keep)
        check(attend(ops, b, **kw), b, **kw)


def test_scratch_is_sound_again_after_an_error_is_read(ops):
    """A call that gave up half way leaves its counts of finished parts behind;
    reading its error word clears them with it."""
    ws = ops.paged_workspace(torch.device("cuda"), 64)
    ws[:1 << 16].view(torch.int32)[64:4096] = 1000  # every counter
    ws[:4].view(torch.int32)[0] = 1
    assert ops.paged_device_error(ws) == 1
    assert ops.paged_device_error(ws) == 0
    for lens in (([1, 2], [9000, 5000]), ([40], [6001])):  # divided and joined
        b = R.Batch(*lens, 8, 1, 64, 64, BF, BF, seed=3)
        check(attend(ops, b, workspace=ws), b)


def test_arguments_elsewhere_are_refused(ops):
    """Scratch, tables and sinks that no kernel on this GPU could read, and
    scratch whose bytes are not what its numel says."""
    b = R.Batch([1], [5], 8, 2, 64, 16, BF, BF)
    n = ops.paged_workspace(torch.device("cuda"), 64).numel()
    t = torch.rand(8, 32, device="cuda")
    qkv = torch.zeros(1, 12 * 64, dtype=BF, device="cuda")
    for ws in (torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8).pin_memory(),
               torch.zeros(n // 4, dtype=torch.float32, device="cuda"),
               torch.zeros(2 * n, dtype=torch.uint8, device="cuda")[::2],
               torch.zeros(1, dtype=torch.uint8, device="cuda").expand(n)):
        with pytest.raises((RuntimeError, ValueError)):
            attend(ops, b, workspace=ws)
        with pytest.raises((RuntimeError, ValueError)):
            ops.paged_kv_store(qkv, t, t, b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8, workspace=ws)
    for name in ("k", "v", "table", "cu", "kv", "sinks", "q"):
        c = R.Batch([1], [5], 8, 2, 64, 16, BF, BF)
        setattr(c, name, getattr(c, name).cpu())
        with pytest.raises((RuntimeError, ValueError)):
            attend(ops, c)
    for kw in (dict(cos=t.cpu()), dict(sin=t.cpu()), dict(q_out=torch.empty(1, 8, 64, dtype=BF))):
        a = dict(cos=t, sin=t) | kw
        with pytest.raises((RuntimeError, ValueError)):
            ops.paged_kv_store(qkv, a.pop("cos"), a.pop("sin"), b.k, b.v, b.table, b.cu, b.kv, n_q_heads=8, **a)


@pytest.mark.parametrize("q_len", [1, 3, 0])
def test_more_sequences_than_a_launch_takes(ops, q_len):
    """Over 512 sequences, which the kernels take in several launches: all of one
    length, or (0) of every length up to 20."""
    n = 700
    q_lens = [q_len or i % 21 for i in range(n)]
    b = R.Batch(q_lens, [q + (13 * i) % 90 for i, q in enumerate(q_lens)], 8, 1, 64, 16, BF, BF, seed=q_len)
    check(attend(ops, b), b)


def test_tables_of_the_widest_kind(ops):
    """Nearly 2^30 positions a sequence in the table (of which few are used): the
    launches take fewer sequences, so that their steps can be counted."""
    page = 1 << 20
    narrow = R.Batch([1] * 70 + [3] * 8 + [40], [60 + i for i in range(79)], 8, 1, 128, 128, BF, E4, seed=2)
    k = torch.zeros(narrow.k.shape[0] * 128 // page + 1, 1, page, 128, dtype=E4, device="cuda")
    v = torch.zeros_like(k)
    table = torch.zeros(79, (1 << 30) // page - 1, dtype=torch.int32, device="cuda")
    got = torch.empty_like(narrow.q)
    for i in range(79):  # one at a time: each has its positions at the start of page 0
        for pool, small in ((k, narrow.k), (v, narrow.v)):
            pool[0, :, :128] = small[int(narrow.table[i, 0])]
            pool[0, :, 128:256] = small[int(narrow.table[i, 1])] if narrow.kv_lens[i] > 128 else 0
        out = ops.paged_attention(narrow.q, k, v, table, narrow.cu, narrow.kv, 40, sinks=narrow.sinks)
        rows = slice(int(narrow.cu[i]), int(narrow.cu[i + 1]))
        got[rows] = out[rows]
    check(got, narrow)


@pytest.mark.parametrize("dtype,held,page", [(BF, "same", 16), (BF, "same", 100), (F16, "same", 24), (BF, "e4m3", 16),
                                             (F16, "e4m3", 1)])
@pytest.mark.parametrize("window,keep", [(1, 3), (37, 4), (128, 140), (1000, 5)])
def test_windows_of_wide_heads(ops, window, keep, dtype, held, page):
    """Windows and first tokens at D = 128, by every way that pages are read."""
    for lens in (RAGGED, ([1, 1, 3, 1], [900, 129, 500, 20]), ([200, 70], [640, 1500])):
        b = R.Batch(*lens, 8, 2, 128, page, dtype, E4 if held == "e4m3" else dtype, seed=window + keep)
        kw = dict(window=window, keep_first=keep)
        check(attend(ops, b, **kw), b, **kw)
