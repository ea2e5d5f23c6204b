"""Log probabilities of given tokens, entropy and alternatives
(qg_logprobs_dev) against the definition in 64 bits.

Tolerances, u = 2^-24: x - m is off by u |x - m|, log Z by the relative error
of Z (a sum of n terms in f32, some hundred one after the other: 2^-16) and by u
log Z, the result by one rounding more; the entropy's terms (x - m) p likewise,
with sum |x - m| p <= H + log n in their place."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NONE = 0xFFFFFFFF


def definition(x):
    """(log probabilities, entropy) of rows [r, n]; f64, NaN where a row has none."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = np.max(x, axis=1, keepdims=True)
        d = x - m
        d[~np.isfinite(m[:, 0])] = np.nan
        e = np.exp(d)
        z = e.sum(1, keepdims=True)
        lp = d - np.log(z)
        ent = np.log(z[:, 0]) - np.where(e > 0, d * e, np.where(np.isnan(e), np.nan, 0)).sum(1) / z[:, 0]
    return lp, ent


def order(x):
    """Ids by value, ties by id, no NaN."""
    ids = np.argsort(-x.astype(np.float64), axis=None, kind="stable")
    return ids[~np.isnan(x[ids])]


def call(ctx, x, tokens=None, k=0, entropy=True, ld=None, off=0):
    import torch
    r, n = x.shape
    ld = ld or n
    buf = torch.full((r * ld + off + 8,), 3.0e4, dtype=torch.float16 if x.dtype == np.float16 else torch.float32, device="cuda")
    d = torch.as_strided(buf, (r, n), (ld, 1), off)
    d.copy_(torch.from_numpy(x).cuda())
    t = None if tokens is None else torch.from_numpy(np.asarray(tokens, np.uint32).view(np.int32)).cuda()
    g = 0 if tokens is None else tokens.shape[1]
    lp = torch.full((r, g), 7.0, device="cuda")
    ent = torch.full((r + 2,), 7.0, device="cuda")
    ids, tl = torch.full((r, k), -7, dtype=torch.int32, device="cuda"), torch.full((r, k), 7.0, device="cuda")
    size = ctx.logprobs_work(r, n, k)
    work = torch.full((size + 64,), 0x55, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.logprobs_dev(d, t, lp if g else None, ent[1:-1] if entropy else None, ids if k else None, tl if k else None, work[:size])
    ctx.synchronize()
    assert bool((work[size:] == 0x55).all()) and float(ent[0]) == 7.0 and float(ent[-1]) == 7.0
    return lp.cpu().numpy(), ent[1:-1].cpu().numpy(), ids.cpu().numpy().view(np.uint32), tl.cpu().numpy()


def close(got, want, tol):
    got = got.astype(np.float64)
    inf = np.isinf(want)
    assert (np.isnan(got) == np.isnan(want)).all()
    assert (got[inf] == want[inf]).all()
    ok = np.isfinite(want)
    bad = np.abs(got[ok] - want[ok]) > tol[ok]
    assert not bad.any(), (np.abs(got[ok] - want[ok]).max(), tol[ok].min())


def check(ctx, x, tokens=None, k=0, first=None, **kw):
    """Every row of a call, or its first ones."""
    lp, ent, ids, tl = call(ctx, x, tokens, k, **kw)
    x, lp, ent, ids, tl = (y[:first] for y in (x, lp, ent, ids, tl))
    tokens = None if tokens is None else tokens[:first]
    wlp, went = definition(x)
    n = x.shape[1]
    # f32 steps of x itself do not enter: they are the operator's input
    near = lambda w: 4 * U * np.abs(w) + 4 * U * np.abs(np.nanmax(np.where(np.isfinite(x), x, 0).astype(np.float64), 1))[:, None] + 2.0 ** -16  # noqa: E731
    if tokens is not None:
        t = tokens.astype(np.int64)
        want = np.where(t < n, np.take_along_axis(wlp, np.minimum(t, n - 1), 1), np.nan)
        want[t == NONE] = 0
        close(lp, want, near(want))
    close(ent, went, 4 * U * np.abs(went) + (went + np.log(n)) * 2.0 ** -15)
    for r in range(len(x) if k else 0):
        want = order(x[r])[:k]
        full = np.full(k, NONE, np.uint32)
        full[:len(want)] = want
        np.testing.assert_array_equal(ids[r], full)
        wt = np.full(k, -np.inf)
        wt[:len(want)] = wlp[r, want]
        big = np.abs(np.max(np.where(np.isfinite(x[r]), x[r], 0).astype(np.float64)))
        close(tl[r], wt, 4 * U * np.abs(wt) + 4 * U * big + 2.0 ** -16)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 1000, 1023, 1025, 4097, 16384, 32001, 50257, 128256, 152064])
def test_sizes(rinf, ctx, n, dtype):
    rng = np.random.default_rng(n)
    r = 3
    x = (rng.standard_normal((r, n)) * 3).astype(dtype)
    x[0, rng.integers(n)] += 15                                  # a confident row
    tokens = rng.integers(0, n, (r, 2)).astype(np.uint32)
    for k in (0, 1, 5, 20, 64):
        check(ctx, x, tokens, k)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 300])
def test_rows(rinf, ctx, rows):
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, 5003)) * 4).astype(np.float32)
    check(ctx, x, rng.integers(0, 5003, (rows, 1)).astype(np.uint32), 8)


@pytest.mark.parametrize("k", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("n", [40, 3000, 130000])
def test_ties_and_orders(rinf, ctx, n, k):
    """Few distinct values, all equal ones, rising and falling rows: equal logits by id."""
    rng = np.random.default_rng(k)
    x = np.stack([rng.integers(0, 4, n), np.zeros(n), np.arange(n) / 512.0, -np.arange(n) / 512.0, -np.abs(np.arange(n) - n // 2) // 3,
                  np.where(np.arange(n) % 2, 0.0, -0.0)]).astype(np.float32)
    check(ctx, x, rng.integers(0, n, (len(x), 1)).astype(np.uint32), k)


def test_long_parts(rinf, ctx):
    """So many rows that one workgroup takes a row, in several pieces of 16384: the alternatives are
    carried from piece to piece, also where every piece is better (rising) or none is (falling)."""
    rng = np.random.default_rng(12)
    rows, n = 600, 40003
    for dtype in (np.float32, np.float16):
        x = (rng.standard_normal((rows, n)) * 3).astype(dtype)
        x[0], x[1] = np.arange(n) / 64.0, -np.arange(n) / 64.0
        x[2], x[3] = 1.0, rng.integers(0, 3, n)
        x[4, :30000], x[5, 16000:] = -np.inf, -np.inf
        x[6], x[7] = -np.inf, np.nan
        x[8, 39000:] += 20
        x[9] = np.nan
        x[9, [5, 17000, 40000]] = -np.inf, 2.0, 1.0
        tokens = rng.integers(0, n, (rows, 1)).astype(np.uint32)
        check(ctx, x, tokens, 64, first=16)
        check(ctx, x, tokens, 3, first=16, ld=n + 1, off=3)


def test_masked(rinf, ctx):
    """-inf, the types' lowest values, one token left, none left, NaN and +inf: each row by itself."""
    rng = np.random.default_rng(4)
    for dtype, n in ((np.float32, 3001), (np.float16, 3001), (np.float32, 70001)):
        x = (rng.standard_normal((10, n)) * 3).astype(dtype)
        x[0, rng.random(n) < 0.9] = -np.inf
        x[1, rng.random(n) < 0.9] = np.finfo(dtype).min
        x[2] = -np.inf
        x[2, 1234] = 5.0
        x[3] = -np.inf
        x[4, 77] = np.nan
        x[5, 99] = np.inf
        x[6] = np.finfo(dtype).min
        x[7] = np.nan
        x[8, :] = np.finfo(dtype).max
        tokens = np.tile(np.array([[1234, 5, 77, NONE, n, NONE - 1]], np.uint32), (10, 1))
        check(ctx, x, tokens, 6)
        check(ctx, x, tokens, 64)


def test_large_differences(rinf, ctx):
    x = np.array([[3e38, -3e38, 0, 1e38], [-3e38, -3.1e38, -3.3e38, -3.4e38], [1e-40, 0, -1e-40, 2e-45]], np.float32)
    lp, ent, ids, tl = call(ctx, x, np.tile(np.arange(4, dtype=np.uint32), (3, 1)), 4)
    assert lp[0, 0] == 0 and (lp[0, 1:] < -1e37).all() and ent[0] == 0
    assert lp[1, 0] == 0 and ent[1] == 0 and (ids[1] == [0, 1, 2, 3]).all()
    np.testing.assert_allclose(lp[2], -np.log(4), rtol=1e-6)
    assert (ids[2] == [0, 3, 1, 2]).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_strides_and_alignment(rinf, ctx, dtype):
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((5, 4099)) * 3).astype(dtype)
    tokens = rng.integers(0, 4099, (5, 3)).astype(np.uint32)
    for ld, off in ((4099, 1), (4100, 0), (4104, 4), (5000, 3), (8192, 5)):
        check(ctx, x, tokens, 5, ld=ld, off=off)


def test_parts(rinf, ctx):
    """Without tokens, without entropy, without alternatives, without anything, without rows."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((3, 500)).astype(np.float32)
    check(ctx, x, None, 4)
    lp, ent, ids, tl = call(ctx, x, rng.integers(0, 500, (3, 1)).astype(np.uint32), 0, entropy=False)
    assert (ent == 7.0).all()
    call(ctx, x, None, 0, entropy=False)
    call(ctx, x[:0], np.zeros((0, 1), np.uint32), 3)


def test_captured_and_deterministic(rinf, ctx):
    import torch
    rng = np.random.default_rng(8)
    x = torch.from_numpy((rng.standard_normal((2, 60000)) * 3).astype(np.float32)).cuda()
    t = torch.from_numpy(rng.integers(0, 60000, (2, 1)).astype(np.int32)).cuda()
    outs = [[torch.zeros(2, 1, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, 20, dtype=torch.int32, device="cuda"),
             torch.zeros(2, 20, device="cuda")] for _ in range(2)]
    works = [torch.zeros(max(16, ctx.logprobs_work(2, 60000, 20)), dtype=torch.uint8, device="cuda") for _ in range(2)]
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        ctx.logprobs_dev(x, t, *outs[0], works[0], stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(5):
        x.copy_(torch.from_numpy((rng.standard_normal((2, 60000)) * 3).astype(np.float32)).cuda())
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ctx.logprobs_dev(x, t, *outs[1], works[1])
        ctx.synchronize()
        assert all(bool((a == b).all()) for a, b in zip(*outs))


def test_refusals(rinf, ctx):
    import ctypes

    import torch
    lib, n = rinf.load_library(), ctypes.c_size_t()
    x, o = torch.zeros(2, 100, device="cuda"), torch.zeros(2, 64, device="cuda")
    p, q = x.data_ptr(), o.data_ptr()
    work = torch.zeros(max(16, ctx.logprobs_work(2, 100, 4)), dtype=torch.uint8, device="cuda")

    def f(x=p, type=0, rows=2, cols=100, ld=100, t=q, g=1, lp=q, ent=q, k=4, ids=q, tl=q):
        return lib.qg_logprobs_dev(ctx.h, x, type, rows, cols, ld, t, g, lp, ent, k, ids, tl, work.data_ptr(), work.numel(), None)

    assert f(type=12) == 2 and f(type=30) == 2
    assert f(x=None) == 1 and f(t=None) == 1 and f(lp=None) == 1 and f(ids=None) == 1 and f(tl=None) == 1
    assert f(x=p + 2) == 1 and f(ent=q + 1) == 1 and f(tl=q + 2) == 1
    assert f(cols=0) == 7 and f(ld=99) == 7 and f(k=65) == 7 and f(cols=1 << 31, ld=1 << 31) == 7 and f(rows=1 << 31) == 7
    assert f(rows=1 << 24) == 7
    assert f(ld=1 << 62) == 7
    assert lib.qg_logprobs_work(ctx.h, 1, 1, 1, None) == 1 and lib.qg_logprobs_work(None, 1, 1, 1, ctypes.byref(n)) == 1
    with pytest.raises(rinf.QgemvError):
        ctx.logprobs_dev(x, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), o[:, :1].contiguous())
    torch.cuda.synchronize()
