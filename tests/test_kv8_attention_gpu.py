"""Attention over the 8-bit KV cache (qg_kv8_attention_dev) against the formula
in 64 bits over the values the cache holds (test_kv8_gpu.quantised).

Tolerances, with u = 2^-24 (an f32 rounding) and a row's A = max over positions
of scale * sum |q k|: a score's error is at most (hd + 8) u A (products and sums
in f32; two f16 pieces of q leave 2^-22 of it), which is the relative error of
its exp; the sums over L positions add (L / 32 + 64) u, exp and the last
rounding a few u, so an output is off by at most
    max |v| (2 (hd + 8) A + L / 32 + 80) u,
plus, with f16 rows, p rounded to f16 (2^-11 max |v|) and the output's own half
step (2^-11 |o|)."""
from __future__ import annotations

import numpy as np
import pytest

from test_kv8_gpu import NP, all_quantised, dev, i32, read, rows, write

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def reference(q, kq, vq, first, window, scale):
    """(outputs, bounds) of one sequence: rows q [n, heads, hd] at positions
    first .. over the values kq, vq [L, kv, hd]; f64."""
    n, heads, hd = q.shape
    L, kv = kq.shape[:2]
    out, tol = np.zeros((n, heads, hd)), np.zeros((n, heads, 1))
    for i in range(n):
        p = first + i
        lo, hi = max(0, p - window + 1) if window else 0, min(p + 1, L)
        if hi <= lo:
            continue
        for h in range(heads):
            g = h // (heads // kv)
            k, v, x = kq[lo:hi, g].astype(np.float64), vq[lo:hi, g].astype(np.float64), q[i, h].astype(np.float64)
            s = k @ x * scale
            with np.errstate(invalid="ignore"):
                e = np.exp(s - s.max())
                out[i, h] = (e @ v) / e.sum()
                a = (np.abs(k) @ np.abs(x)).max() * abs(scale)
                tol[i, h] = np.abs(v).max() * (2 * (hd + 8) * a + (hi - lo) / 32 + 80) * U
    return out, tol


def run(ctx, cache, q, lens, starts=None, window=0, scale=None, guard=2):
    """The operator's outputs, behind and before rows that have to stay."""
    import torch
    n, heads, hd = q.shape
    buf = torch.full((n + 2 * guard, heads, hd), 7.0, dtype=torch.float32 if q.dtype == np.float32 else torch.float16, device="cuda")
    bytes_ = cache.attention_work(n, heads)
    work = torch.full((max(bytes_, 16) + 64,), 0x55, dtype=torch.uint8, device="cuda")
    dq, dl, ds = dev(q), i32(lens), None if starts is None else i32(starts)
    torch.cuda.synchronize()
    cache.attention_dev(dq, buf[guard:guard + n], dl, work[:bytes_], ds, scale=scale, window=window)
    ctx.synchronize()
    assert bool((work[bytes_:] == 0x55).all())
    got = buf.cpu().numpy()
    assert (got[:guard] == 7.0).all() and (got[n + guard:] == 7.0).all()
    return got[guard:guard + n]


def compare(got, want, tol, f16):
    got = got.astype(np.float64)
    assert (np.isnan(got) == np.isnan(want)).all()
    if f16:
        tol = tol + 2.0 ** -11 * (np.abs(want) + np.abs(want).max(initial=0) * 4)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.nanmax(np.abs(got - want)), np.nanmin(tol))


def case(rinf, ctx, old, new, heads, kv, hd, dtype="f32", window=0, seed=0, scale=None, most=None):
    """Sequences of old[s] cached tokens and new[s] rows, every row checked."""
    rng = np.random.default_rng(seed)
    total = [a + b for a, b in zip(old, new)]
    cache = ctx.kv8(len(old), kv, hd, most or max(total + [1]))
    k = [rows(rng, n, kv, hd, dtype) for n in total]
    v = [rows(rng, n, kv, hd, dtype) for n in total]
    write(ctx, cache, k, v, total)
    q = (rng.standard_normal((sum(new), heads, hd)) * 0.5).astype(NP[dtype])
    starts = np.concatenate([[0], np.cumsum(new)])
    single = all(n == 1 for n in new)
    got = run(ctx, cache, q, total, None if single else starts, window, scale)
    for s in range(len(old)):
        want, tol = reference(q[starts[s]:starts[s + 1]], all_quantised(k[s].astype(np.float32)),
                              all_quantised(v[s].astype(np.float32)), old[s], window, hd ** -0.5 if scale is None else scale)
        compare(got[starts[s]:starts[s + 1]], want, tol, dtype == "f16")
    if single:                                    # the same with starts
        again = run(ctx, cache, q, total, starts, window, scale)
        for s in range(len(old)):
            want, tol = reference(q[s:s + 1], all_quantised(k[s].astype(np.float32)), all_quantised(v[s].astype(np.float32)),
                                  old[s], window, hd ** -0.5 if scale is None else scale)
            compare(again[s:s + 1], want, tol, dtype == "f16")
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (7, 1, 128), (8, 8, 128), (8, 2, 256), (3, 1, 80), (4, 2, 40), (2, 1, 1),
                                         (20, 1, 64), (6, 2, 192), (2, 2, 255), (40, 1, 96)])
def test_steps(rinf, ctx, heads, kv, hd, dtype):
    """One row per sequence, lengths around the ends of blocks and tiles."""
    case(rinf, ctx, [0, 1, 14, 30, 31, 32, 33, 62, 63, 64, 100, 127, 128, 129, 300], [1] * 15, heads, kv, hd, dtype, seed=hd + heads)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (7, 1, 128), (3, 3, 128), (2, 1, 256), (5, 1, 80), (2, 2, 40), (17, 1, 64)])
def test_prompts(rinf, ctx, heads, kv, hd, dtype):
    """Ragged prompts, some of them on top of cached tokens, one with no rows."""
    case(rinf, ctx, [0, 0, 40, 100, 7, 0, 64], [1, 33, 65, 2, 0, 130, 31], heads, kv, hd, dtype, seed=hd + heads)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 50, 64, 129, 4096])
def test_window(rinf, ctx, window, dtype):
    case(rinf, ctx, [0, 90, 200], [70, 1, 40], 4, 2, 64, dtype, window, seed=window)
    case(rinf, ctx, [0, 90, 200, 33], [1] * 4, 4, 2, 128, dtype, window, seed=window)


def test_long(rinf, ctx):
    """Long caches, where the positions are split: one sequence, and a few with very different lengths."""
    case(rinf, ctx, [20000], [1], 4, 1, 128, "f32", seed=1)
    case(rinf, ctx, [9000, 3, 5000, 0], [1] * 4, 8, 2, 64, "f16", seed=2)
    case(rinf, ctx, [6000, 0, 2500], [5, 17, 3], 8, 2, 64, "f32", seed=3)
    case(rinf, ctx, [7000], [3], 4, 1, 128, "f16", window=3000, seed=4)


def test_many_sequences(rinf, ctx):
    rng = np.random.default_rng(3)
    case(rinf, ctx, [int(n) for n in rng.integers(0, 90, 150)], [int(n) for n in rng.integers(0, 4, 150)], 4, 2, 64, "f32", seed=5)
    case(rinf, ctx, [int(n) for n in rng.integers(0, 90, 200)], [1] * 200, 4, 1, 64, "f16", seed=6)


def test_many_groups_of_sequences(rinf, ctx):
    """More sequences than a wave looks at together, a workgroup's items in several of those groups."""
    rng = np.random.default_rng(13)
    case(rinf, ctx, [int(n) for n in rng.integers(0, 40, 1300)], [int(n) for n in rng.integers(0, 3, 1300)], 2, 1, 16, "f32", seed=7)
    case(rinf, ctx, [int(n) for n in rng.integers(0, 40, 1100)], [1] * 1100, 1, 1, 16, "f16", seed=8)


@pytest.mark.parametrize("heads,n", [(1, 20), (1, 100), (512, 130)])
def test_f32_has_both_pieces(rinf, ctx, heads, n):
    """f32 rows against a bound so narrow that a lost low piece of q or of p is
    past it (tiles of 16, 64 and 128 pairs).  A row has two elements that are not
    zero, so that its scores add two products (the others add exactly nothing):
    the bound of `reference` with 2 for hd, over at most 130 positions."""
    rng = np.random.default_rng(heads + n)
    hd, nz = 64, 2
    cache = ctx.kv8(1, heads, hd, n)
    k, v = (rng.standard_normal((n, heads, hd)).astype(np.float32) for _ in range(2))
    write(ctx, cache, [k], [v], [n])
    q = np.zeros((n, heads, hd), np.float32)
    for h in range(heads):
        q[:, h, rng.permutation(hd)[:nz]] = rng.uniform(3, 5, (n, nz)) * rng.choice([-1, 1], (n, nz))
    got = run(ctx, cache, q, [n], [0, n], scale=1.0).astype(np.float64)
    kq, vq = all_quantised(k).astype(np.float64), all_quantised(v).astype(np.float64)
    sees = np.tril(np.ones((n, n), bool))
    past = np.zeros(2)
    some = range(heads) if heads == 1 else range(0, heads, 37)

    def out(x, h, rounded):
        s = np.where(sees, x @ kq[:, h].T, -np.inf)
        e = np.exp(s - s.max(1, keepdims=True))
        p = e.astype(np.float16).astype(np.float64) if rounded else e
        return p @ vq[:, h] / e.sum(1, keepdims=True), s

    for h in some:
        x = q[:, h].astype(np.float64)
        want, s = out(x, h, False)
        a = (np.abs(x) @ np.abs(kq[:, h]).T * sees).max(1, keepdims=True)
        tol = np.abs(vq[:, h]).max() * (2 * (nz + 8) * a + n / 32 + 80) * U
        assert (np.abs(got[:, h] - want) <= tol).all(), (h, (np.abs(got[:, h] - want) / tol).max())
        past[0] += (np.abs(out(x.astype(np.float16).astype(np.float64), h, False)[0] - want) > tol).any(1).mean()
        past[1] += (np.abs(out(x, h, True)[0] - want) > tol).any(1).mean()
    # without either low piece rows would be past their bounds (one is enough to
    # fail; a row that sees one position hides its score, and here the largest
    # weight, 1, has no low piece)
    assert (past > 0).all(), past
    cache.free()


def test_scales(rinf, ctx):
    """Scores that spread far, that all are equal, and a negative scale."""
    for scale in (0.0, 1.0, -0.3, 30.0):
        case(rinf, ctx, [0, 70], [40, 3], 4, 2, 64, "f32", scale=scale, seed=8)
        case(rinf, ctx, [200, 70], [1, 1], 4, 2, 64, "f32", scale=scale, seed=9)


def test_large_and_small_values(rinf, ctx):
    """q and v of any size that f32 sums take: the pieces of q are scaled by row."""
    rng = np.random.default_rng(14)
    for qs, ks, vs in ((1e-20, 1e20, 1e30), (1e18, 1e-18, 1e-30), (1e-3, 1e3, 1.0)):
        cache = ctx.kv8(1, 1, 64, 128)
        k, v = rows(rng, 100, 1, 64, scale=ks), rows(rng, 100, 1, 64, scale=vs)
        write(ctx, cache, [k], [v], [100])
        q = (rng.standard_normal((30, 4, 64)) * qs).astype(np.float32)
        got = run(ctx, cache, q, [100], [0, 30])
        want, tol = reference(q, all_quantised(k), all_quantised(v), 70, 0, 0.125)
        compare(got, want, tol, False)
        cache.free()


def test_rows_that_see_nothing(rinf, ctx):
    """Rows before position 0 give zeros, rows past the cache what there is; an empty sequence, and no rows at all."""
    rng = np.random.default_rng(15)
    kv, hd, heads = 2, 64, 4
    k, v = rows(rng, 64, kv, hd), rows(rng, 64, kv, hd)
    cache = ctx.kv8(2, kv, hd, 64)
    write(ctx, cache, [k, k[:0]], [v, v[:0]], [64, 0])
    kq, vq = all_quantised(k), all_quantised(v)
    q = rng.standard_normal((20, heads, hd)).astype(np.float32)
    got = run(ctx, cache, q, [5, 0], [0, 12, 20])            # positions -7 .. 4, and -8 .. -1
    want, tol = reference(q[:12], kq[:5], vq[:5], -7, 0, 0.125)
    compare(got[:12], want, tol, False)
    assert (got[:7] == 0).all() and (got[12:] == 0).all()
    got = run(ctx, cache, q[:2], [70, 0])                     # single rows: past the cache, and of an empty sequence
    want, tol = reference(q[:1], kq, vq, 69, 0, 0.125)
    compare(got[:1], want, tol, False)
    assert (got[1] == 0).all()
    got = run(ctx, cache, q[:12], [70, 0], [0, 12, 12], window=3)    # positions 58 .. 69 of 64, three each
    want, tol = reference(q[:12], kq, vq, 58, 3, 0.125)
    compare(got, want, tol, False)
    assert (got[8:] == 0).all()
    got = run(ctx, cache, q, [64, 64], [0, 5, 8])             # rows behind the last sequence stay
    assert (got[8:] == 7.0).all()
    assert run(ctx, cache, q[:0], [64, 64], [0, 0, 0]).shape[0] == 0
    cache.free()


def test_non_finite_out_of_sight(rinf, ctx):
    """NaN and infinite blocks reach only the rows and heads that see them; stale positions reach none."""
    rng = np.random.default_rng(16)
    kv, hd, heads, n = 2, 64, 4, 130
    for what in (np.nan, np.inf):
        for which in ("k", "v"):
            k, v = rows(rng, n, kv, hd), rows(rng, n, kv, hd)
            (k if which == "k" else v)[70, 1, 3] = what           # block 2 of head 1
            cache = ctx.kv8(1, kv, hd, 256)
            write(ctx, cache, [k], [v], [n])
            q = rng.standard_normal((n, heads, hd)).astype(np.float32)
            got = run(ctx, cache, q, [n], [0, n])
            want, tol = reference(q, all_quantised(k), all_quantised(v), 0, 0, 0.125)
            assert np.isnan(want[64:, 2:]).all() and np.isfinite(want[:, :2]).all() and np.isfinite(want[:64]).all()
            compare(got, want, tol, False)
            got = run(ctx, cache, q, [n], [0, n], window=20)        # seen again no more from position 115 on
            want, tol = reference(q, all_quantised(k), all_quantised(v), 0, 20, 0.125)
            compare(got, want, tol, False)
            assert np.isfinite(got[115:]).all()
            # a shorter conversation over it: the NaN block lies behind its end
            write(ctx, cache, [k[:40]], [v[:40]], [40])
            got = run(ctx, cache, q[:1], [40])
            want, tol = reference(q[:1], all_quantised(k[:40]), all_quantised(v[:40]), 39, 0, 0.125)
            compare(got, want, tol, False)
            cache.free()
    q = rng.standard_normal((3, heads, hd)).astype(np.float32)       # a row of q that is not finite: its own alone
    q[1, 2, 5] = np.nan
    cache = ctx.kv8(1, kv, hd, 64)
    k, v = rows(rng, 50, kv, hd), rows(rng, 50, kv, hd)
    write(ctx, cache, [k], [v], [50])
    got = run(ctx, cache, q, [50], [0, 3])
    assert np.isnan(got[1, 2]).all()
    got[1, 2] = 0
    assert np.isfinite(got).all()
    cache.free()


def test_strides_and_types(rinf, ctx):
    """q and out inside wider buffers, heads before rows, and not aligned to 16 bytes."""
    import torch
    rng = np.random.default_rng(17)
    kv, hd, heads, n = 2, 64, 4, 40
    k, v = rows(rng, 90, kv, hd), rows(rng, 90, kv, hd)
    cache = ctx.kv8(1, kv, hd, 96)
    write(ctx, cache, [k], [v], [90])
    for t in ("f32", "f16"):
        q = rng.standard_normal((n, heads, hd)).astype(NP[t])
        want, tol = reference(q, all_quantised(k), all_quantised(v), 50, 0, 0.125)
        tt = torch.float32 if t == "f32" else torch.float16
        lens, starts = i32([90]), i32([0, n])
        work = torch.zeros(max(16, cache.attention_work(n, heads)), dtype=torch.uint8, device="cuda")
        for make in (lambda: torch.zeros(heads, n, hd, dtype=tt, device="cuda").permute(1, 0, 2),
                     lambda: torch.zeros(n, heads + 3, hd, dtype=tt, device="cuda")[:, 1:1 + heads],
                     lambda: torch.zeros(n * heads * hd + 1, dtype=tt, device="cuda")[1:].view(n, heads, hd),
                     lambda: torch.zeros(n, heads, hd + 5, dtype=tt, device="cuda")[:, :, :hd]):
            dq, out = make(), make()
            dq.copy_(dev(q))
            torch.cuda.synchronize()
            cache.attention_dev(dq, out, lens, work, starts)
            ctx.synchronize()
            compare(out.cpu().numpy(), want, tol, t == "f16")
    cache.free()


def test_deterministic_and_on_another_stream(rinf, ctx):
    """The same call gives the same bits, alone, beside others on other streams with workspaces of their own, and
    in a captured graph that is replayed as lengths change."""
    import torch
    rng = np.random.default_rng(18)
    kv, hd, heads, n0 = 2, 128, 8, 3000
    cache = ctx.kv8(2, kv, hd, 4096)
    k, v = rows(rng, n0, kv, hd), rows(rng, n0, kv, hd)
    write(ctx, cache, [k, k[:77]], [v, v[:77]], [n0, 77])
    q = dev(rng.standard_normal((2, heads, hd)).astype(np.float32))
    size = max(16, cache.attention_work(2, heads))
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros(2, heads, hd, device="cuda") for _ in range(4)]
    works = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(4)]
    lens = i32([n0, 77])
    torch.cuda.synchronize()
    for rep in range(5):
        for s, o, w in zip(streams, outs, works):
            cache.attention_dev(q, o, lens, w, stream=s.cuda_stream)
        cache.attention_dev(q, outs[3], lens, works[3])
        torch.cuda.synchronize()
        ctx.synchronize()
        assert all(bool((o == outs[0]).all()) for o in outs)
    g = torch.cuda.CUDAGraph()
    out = torch.zeros(2, heads, hd, device="cuda")
    with torch.cuda.graph(g, stream=streams[0]):
        cache.attention_dev(q, out, lens, works[0], stream=torch.cuda.current_stream().cuda_stream)
    for m in (n0, 1, 32, 1500, 0, n0):
        lens.copy_(i32([m, min(m, 77)]))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        cache.attention_dev(q, outs[1], lens, works[1], stream=streams[1].cuda_stream)
        torch.cuda.synchronize()
        assert bool((out == outs[1]).all())
    cache.free()


def test_write_then_attend(rinf, ctx):
    """A conversation as it is used: a prompt, steps, write and attention together, checked at every step."""
    import torch
    rng = np.random.default_rng(19)
    kv, hd, heads = 2, 64, 6
    cache = ctx.kv8(2, kv, hd, 200)
    hk, hv = [np.zeros((0, kv, hd), np.float32)] * 2, [np.zeros((0, kv, hd), np.float32)] * 2
    work = torch.zeros(max(16, cache.attention_work(128, heads)), dtype=torch.uint8, device="cuda")
    for n in ([40, 3], [1, 1], [1, 1], [30, 60], [1, 0], [1, 1], [5, 2]):
        k, v = ([rows(rng, m, kv, hd) for m in n] for _ in range(2))
        hk, hv = ([np.concatenate([a, b]) for a, b in zip(h, x)] for h, x in ((hk, k), (hv, v)))
        q = rng.standard_normal((sum(n), heads, hd)).astype(np.float32)
        starts, lens = np.concatenate([[0], np.cumsum(n)]), [len(h) for h in hk]
        dk, dv, dq = dev(np.concatenate(k)), dev(np.concatenate(v)), dev(q)
        out, ds, dl = torch.zeros_like(dq), i32(starts), i32(lens)
        torch.cuda.synchronize()
        cache.write_dev(dk, dv, dl, ds)
        cache.attention_dev(dq, out, dl, work, ds)
        ctx.synchronize()
        for s in range(2):
            want, tol = reference(q[starts[s]:starts[s + 1]], all_quantised(hk[s]), all_quantised(hv[s]), lens[s] - n[s], 0, hd ** -0.5)
            compare(out.cpu().numpy()[starts[s]:starts[s + 1]], want, tol, False)
    cache.free()


@pytest.mark.parametrize("rows_each", [1, 45])
def test_captured_step_of_a_batch(rinf, ctx, rows_each):
    """Write, attention and log probabilities as one captured step of a batch; between the replays the
    lengths, the split of the rows and the tokens change, and eager calls run on the same cache."""
    import torch
    rng = np.random.default_rng(23 + rows_each)
    kv, hd, heads, seqs, most = 2, 64, 4, 3, 400
    n = rows_each * seqs
    cache = ctx.kv8(seqs, kv, hd, most)
    f32, dev0 = torch.float32, "cuda"
    k, v = torch.zeros(n, kv, hd, device=dev0), torch.zeros(n, kv, hd, device=dev0)
    q, out = torch.zeros(n, heads, hd, device=dev0), torch.zeros(n, heads, hd, device=dev0)
    lens, starts = i32([0] * seqs), i32([0] * (seqs + 1))
    ids = torch.zeros(n, 1, dtype=torch.int32, device=dev0)
    lp, ent, tids, tlp = (torch.zeros(n, c, dtype=d, device=dev0) for c, d in ((1, f32), (1, f32), (5, torch.int32), (5, f32)))
    work = torch.zeros(max(16, cache.attention_work(n, heads)), dtype=torch.uint8, device=dev0)
    lwork = torch.zeros(max(16, ctx.logprobs_work(n, heads * hd, 5)), dtype=torch.uint8, device=dev0)
    torch.cuda.synchronize()

    def step(stream):
        cache.write_dev(k, v, lens, starts, stream=stream)
        cache.attention_dev(q, out, lens, work, starts, stream=stream)
        ctx.logprobs_dev(out.view(n, heads * hd), ids, lp, ent, tids, tlp, lwork, stream=stream)

    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        step(torch.cuda.current_stream().cuda_stream)
    hk, hv = ([np.zeros((0, kv, hd), np.float32)] * seqs for _ in range(2))
    for turn in range(5):
        m = [rows_each] * seqs if rows_each == 1 else [int(x) for x in rng.multinomial(n - turn, [0.5, 0.1, 0.4])]
        nk, nv = ([rows(rng, x, kv, hd) for x in m] for _ in range(2))
        hk, hv = ([np.concatenate([a, b]) for a, b in zip(h, x)] for h, x in ((hk, nk), (hv, nv)))
        total, at = [len(h) for h in hk], np.concatenate([[0], np.cumsum(m)])
        hq, given = rng.standard_normal((n, heads, hd)).astype(np.float32), rng.integers(0, heads * hd, (n, 1))
        k[:at[-1]].copy_(dev(np.concatenate(nk))), v[:at[-1]].copy_(dev(np.concatenate(nv))), q.copy_(dev(hq))
        lens.copy_(i32(total)), starts.copy_(i32(at)), ids.copy_(i32(given)), out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay() if turn % 2 == 0 else step(st.cuda_stream)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert (got[at[-1]:] == 7.0).all()
        for s in range(seqs):
            want, tol = reference(hq[at[s]:at[s + 1]], all_quantised(hk[s]), all_quantised(hv[s]), total[s] - m[s], 0, hd ** -0.5)
            compare(got[at[s]:at[s + 1]], want, tol, False)
        x = got.reshape(n, heads * hd).astype(np.float64)
        p = x - x.max(1, keepdims=True)
        p -= np.log(np.exp(p).sum(1, keepdims=True))
        # 256 terms: sums and exponents within 300 steps of 2^-24
        assert np.abs(lp.cpu().numpy() - np.take_along_axis(p, given, 1)).max() < 300 * U * np.abs(p).max()
        order = np.argsort(-x, axis=1, kind="stable")[:, :5]
        assert (tids.cpu().numpy() == order).all()
    cache.free()


def test_offsets_past_32_bits(rinf, ctx):
    """The end of a cache whose codes lie past 4 GB, by single rows and by many."""
    rng = np.random.default_rng(29)
    kv, hd, heads, most, n = 4, 256, 8, 1 << 20, 40
    cache = ctx.kv8(3, kv, hd, most)
    assert cache.nbytes > 6 << 30
    k, v = rows(rng, n, kv, hd), rows(rng, n, kv, hd)
    none = np.zeros((0, kv, hd), np.float32)
    write(ctx, cache, [none, none, k], [none, none, v], [0, 0, most])
    zeros = np.zeros((24, kv, hd), np.float32)                # the 24 positions of its block before them
    kq, vq = all_quantised(np.concatenate([zeros, k])), all_quantised(np.concatenate([zeros, v]))
    gk, gv = read(ctx, cache, 2, most - 64, 64)
    np.testing.assert_array_equal(gk, kq)
    np.testing.assert_array_equal(gv, vq)
    for m in (1, n):
        q = rng.standard_normal((m, heads, hd)).astype(np.float32)
        got = run(ctx, cache, q, [0, 0, most], [0, 0, 0, m], window=24)
        want, tol = reference(q, kq, vq, 64 - m, 24, hd ** -0.5)
        compare(got, want, tol, False)
    cache.free()


def test_refusals(rinf, ctx):
    import ctypes

    import torch
    lib = rinf.load_library()
    cache = ctx.kv8(2, 2, 64, 64)
    q, out, lens = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda"), i32([1, 1])
    n = ctypes.c_size_t()
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 2, 4, ctypes.byref(n)) == 0
    work = torch.zeros(max(16, n.value), dtype=torch.uint8, device="cuda")

    def call(heads=4, rq=None, ro=None, w=work.data_ptr(), size=work.numel(), b=None):
        rq = rq or rinf.Rows(q.data_ptr(), 0, 256, 64)
        ro = ro or rinf.Rows(out.data_ptr(), 0, 256, 64)
        b = b or rinf.Batch(2, None, lens.data_ptr())
        return lib.qg_kv8_attention_dev(ctx.h, cache.h, ctypes.byref(b), heads, ctypes.byref(rq), 0.125, 0, ctypes.byref(ro),
                                        w, size, None)

    assert call() == 0
    assert call(heads=3) == 7 and call(heads=0) == 7
    assert call(rq=rinf.Rows(q.data_ptr(), 1, 256, 64)) == 2 and call(rq=rinf.Rows(q.data_ptr(), 8, 256, 64)) == 2
    assert call(ro=rinf.Rows(out.data_ptr(), 0, 64, 64)) == 7 and call(ro=rinf.Rows(out.data_ptr(), 0, 0, 64)) == 7
    assert call(rq=rinf.Rows(None, 0, 256, 64)) == 1 and call(ro=rinf.Rows(out.data_ptr() + 1, 0, 256, 64)) == 1
    assert call(b=rinf.Batch(1, None, lens.data_ptr())) == 7 and call(b=rinf.Batch(2, None, None)) == 1
    if n.value:
        assert call(size=n.value - 1) == 7 and call(w=None) == 1 and call(w=work.data_ptr() + 4) == 1
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 2, 3, ctypes.byref(n)) == 7
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 1 << 31, 4, ctypes.byref(n)) == 7
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 1 << 28, 2, ctypes.byref(n)) == 7
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 1 << 27, 16, ctypes.byref(n)) == 7       # 2^31 rows of heads
    assert call(b=rinf.Batch(1 << 28, lens.data_ptr(), lens.data_ptr()), ro=rinf.Rows(out.data_ptr(), 0, 256, 64)) == 7
    assert call(heads=16, b=rinf.Batch(1 << 27, lens.data_ptr(), lens.data_ptr()), ro=rinf.Rows(out.data_ptr(), 0, 1024, 64)) == 7
    assert lib.qg_kv8_attention_work(ctx.h, cache.h, 2, 4, None) == 1
    torch.cuda.synchronize()
    cache.free()
