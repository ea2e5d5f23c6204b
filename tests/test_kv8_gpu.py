"""The 8-bit KV cache (qg_kv8_write_dev, qg_kv8_read_dev) against its
definition in 64 bits: blocks of 32 positions, scale = max |x| / 127 in f32,
codes x / scale to the nearest with ties to even.  What is read back is held to
the definition bit for bit (code * scale rounded once to f32, then to the
output's type), whatever the calls the tokens came in."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B = 32
NP = {"f32": np.float32, "f16": np.float16}


def quantised(x):
    """Values of one head's positions [n, hd] (float32) as the cache holds them."""
    out = np.zeros_like(x, dtype=np.float32)
    for b in range(0, len(x), B):
        y = x[b:b + B].astype(np.float64)
        if not np.isfinite(y).all():
            out[b:b + B] = np.nan
            continue
        s = np.float32(np.abs(y).max() / 127)
        if s >= 2.0 ** -126:
            out[b:b + B] = np.round(y / np.float64(s)).astype(np.float32) * s
    return out


def all_quantised(x):
    """[n, heads, hd]"""
    return np.stack([quantised(x[:, h]) for h in range(x.shape[1])], 1) if len(x) else x.astype(np.float32)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return dev(np.asarray(a, dtype=np.uint32).view(np.int32))


def write(ctx, cache, ks, vs, lens, single=False):
    """One call: ks, vs: per sequence the new rows [n, heads, hd]."""
    import torch
    starts = np.concatenate([[0], np.cumsum([len(k) for k in ks])])
    k, v = dev(np.concatenate(ks)), dev(np.concatenate(vs))
    d_lens, d_starts = i32(lens), None if single else i32(starts)
    torch.cuda.synchronize()
    cache.write_dev(k, v, d_lens, d_starts)
    ctx.synchronize()


def read(ctx, cache, seq, pos, n, dtype="f32", n_seqs=1):
    import torch
    shape = (n_seqs * n, cache.n_kv_heads, cache.head_dim)
    t = torch.float32 if dtype == "f32" else torch.float16
    k, v = torch.full(shape, 7.0, dtype=t, device="cuda"), torch.full(shape, 7.0, dtype=t, device="cuda")
    torch.cuda.synchronize()
    cache.read_dev(seq, n_seqs, pos, n, k, v)
    ctx.synchronize()
    return k.cpu().numpy(), v.cpu().numpy()


def rows(rng, n, heads, hd, dtype="f32", scale=1.0):
    x = rng.standard_normal((n, heads, hd)) * scale
    # magnitudes that keep growing and shrinking: the scale of an open block changes often
    return (x * np.exp2(rng.integers(-3, 4, (n, heads, 1)))).astype(NP[dtype])


def check(ctx, cache, hist_k, hist_v):
    for s, (hk, hv) in enumerate(zip(hist_k, hist_v)):
        if not len(hk):
            continue
        k, v = read(ctx, cache, s, 0, len(hk))
        np.testing.assert_array_equal(k, all_quantised(hk.astype(np.float32)))
        np.testing.assert_array_equal(v, all_quantised(hv.astype(np.float32)))


@pytest.mark.parametrize("hd", [1, 3, 16, 40, 64, 80, 96, 128, 192, 255, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_prompt_and_steps(rinf, ctx, hd, dtype):
    """A ragged prompt, then steps across two block ends: every length is the definition's."""
    rng = np.random.default_rng(hd)
    heads, seqs = 2, 3
    cache = ctx.kv8(seqs, heads, hd, 160)
    first = [0, 45, 64]
    hk = [rows(rng, n, heads, hd, dtype) for n in first]
    hv = [rows(rng, n, heads, hd, dtype) for n in first]
    write(ctx, cache, hk, hv, first)
    check(ctx, cache, hk, hv)
    for step in range(40):
        k = [rows(rng, 1, heads, hd, dtype) for _ in range(seqs)]
        v = [rows(rng, 1, heads, hd, dtype) for _ in range(seqs)]
        hk, hv = ([np.concatenate([a, b]) for a, b in zip(h, x)] for h, x in ((hk, k), (hv, v)))
        write(ctx, cache, k, v, [len(h) for h in hk], single=True)
        if step % 7 == 0 or step > 30:
            check(ctx, cache, hk, hv)
    check(ctx, cache, hk, hv)
    cache.free()


@pytest.mark.parametrize("hd,heads,dtype", [(16, 40, "f32"), (5, 48, "f16"), (128, 33, "f16"), (200, 33, "f32"), (64, 64, "f16")])
def test_long_prompts(rinf, ctx, hd, heads, dtype):
    """More blocks than workgroups fit, so that one takes several: prompts of all
    remainders, then more rows from inside a block on; a NaN and zeros in the middle."""
    rng = np.random.default_rng(hd)
    first, then = [700, 129, 0, 384, 33], [1, 450, 320, 0, 95]
    total = [a + b for a, b in zip(first, then)]
    cache = ctx.kv8(len(total), heads, hd, max(total))
    hk = [rows(rng, n, heads, hd, dtype) for n in total]
    hv = [rows(rng, n, heads, hd, dtype) for n in total]
    hk[0][333, 1, hd - 1], hv[1][200, 2, 0] = np.nan, np.inf
    hk[0][96:160, 3], hv[2][64:96, 4] = 0, 0
    for call in range(2):
        k, v = ([x[:a] if call == 0 else x[a:] for x, a in zip(h, first)] for h in (hk, hv))
        write(ctx, cache, k, v, first if call == 0 else total)
        check(ctx, cache, *([x[:a] for x, a in zip(h, first)] if call == 0 else h for h in (hk, hv)))
    cache.free()


@pytest.mark.parametrize("seed", range(4))
def test_any_calls_give_one_cache(rinf, ctx, seed):
    """Calls of 0 to 100 rows a sequence, in any ragged mix."""
    rng = np.random.default_rng(seed)
    seqs, heads, hd, most = int(rng.integers(1, 70)), int(rng.integers(1, 4)), 64, 400
    cache = ctx.kv8(seqs, heads, hd, most)
    hk = [np.zeros((0, heads, hd), np.float32) for _ in range(seqs)]
    hv = [np.zeros((0, heads, hd), np.float32) for _ in range(seqs)]
    for _ in range(8):
        n = [min(most - len(h), int(rng.choice([0, 0, 1, 1, 5, 31, 32, 33, 64, 100]))) for h in hk]
        k, v = ([rows(rng, m, heads, hd) for m in n] for _ in range(2))
        hk, hv = ([np.concatenate([a, b]) for a, b in zip(h, x)] for h, x in ((hk, k), (hv, v)))
        write(ctx, cache, k, v, [len(h) for h in hk])
    check(ctx, cache, hk, hv)
    cache.free()


def test_back_and_again(rinf, ctx):
    """The last call once more gives the same cache; so does another one from
    the same position or inside the block that was open before it."""
    rng = np.random.default_rng(5)
    heads, hd = 2, 64
    base = [rows(rng, 40, heads, hd), rows(rng, 40, heads, hd)]
    for n, back, m in ((70, 0, 70), (70, 0, 3), (5, 0, 5), (70, 6, 20), (60, 8, 90), (24, 0, 24), (24, 3, 24), (100, 0, 24)):
        cache = ctx.kv8(1, heads, hd, 256)
        write(ctx, cache, [base[0]], [base[1]], [40])
        x = [rows(rng, n, heads, hd, scale=2.0) for _ in range(2)]
        write(ctx, cache, [x[0]], [x[1]], [40 + n])
        write(ctx, cache, [x[0]], [x[1]], [40 + n])
        check(ctx, cache, [np.concatenate([base[0], x[0]])], [np.concatenate([base[1], x[1]])])
        y = [rows(rng, m, heads, hd, scale=0.5) for _ in range(2)]
        write(ctx, cache, [y[0]], [y[1]], [40 - back + m])
        check(ctx, cache, [np.concatenate([base[0][:40 - back], y[0]])], [np.concatenate([base[1][:40 - back], y[1]])])
        cache.free()


def test_far_back(rinf, ctx):
    """Back into a block whose f32 values are gone: its earlier positions go on
    with their 8-bit values, in later steps too."""
    rng = np.random.default_rng(6)
    heads, hd = 2, 128
    x = [rows(rng, 200, heads, hd) for _ in range(2)]
    cache = ctx.kv8(1, heads, hd, 256)
    write(ctx, cache, [x[0]], [x[1]], [200])
    kept = [all_quantised(a)[:50] for a in x]           # as the full blocks hold them
    y = [rows(rng, 3, heads, hd) for _ in range(2)]
    hist = [np.concatenate([a, b]) for a, b in zip(kept, y)]
    write(ctx, cache, [y[0]], [y[1]], [53])
    check(ctx, cache, [hist[0]], [hist[1]])
    for _ in range(20):
        y = [rows(rng, 1, heads, hd) for _ in range(2)]
        hist = [np.concatenate([a, b]) for a, b in zip(hist, y)]
        write(ctx, cache, [y[0]], [y[1]], [len(hist[0])])
        check(ctx, cache, [hist[0]], [hist[1]])
    # a new conversation in the same place
    z = [rows(rng, 70, heads, hd) for _ in range(2)]
    write(ctx, cache, [z[0]], [z[1]], [70])
    check(ctx, cache, [z[0]], [z[1]])
    cache.free()


def test_values_next_to_a_border(rinf, ctx):
    """Quotients on and next to a half (scale 2^-5 and scales that are no power of two), the f32's
    smallest scales, zeros: the code is the nearest, ties to even."""
    rng = np.random.default_rng(7)
    heads, hd, n = 4, 128, 64
    x = np.zeros((n, heads, hd), np.float32)
    x[:, 0] = rng.integers(-253, 254, (n, hd)) / 64.0                # ties
    x[::32, 0, 0] = 127 / 32.0
    s = np.float32(0.0371)
    for t in range(n):
        half = (rng.integers(-126, 126, hd) + 0.5).astype(np.float64) * np.float64(s)
        y = half.astype(np.float32)
        up = rng.integers(-2, 3, hd)
        for _ in range(2):
            y = np.where(up > 0, np.nextafter(y, np.float32(np.inf)), np.where(up < 0, np.nextafter(y, np.float32(-np.inf)), y))
            up = up - np.sign(up)
        x[t, 1] = y
    x[::32, 1, 0] = s * np.float32(127)
    x[:, 2] = rng.standard_normal((n, hd)) * 2.0 ** -118             # scales around 2^-126
    x[:32, 2] *= 2.0 ** -4
    cache = ctx.kv8(1, heads, hd, n)
    write(ctx, cache, [x], [x[:, ::-1].copy()], [n])
    check(ctx, cache, [x], [x[:, ::-1].copy()])
    cache.free()


def test_large_values_and_non_finite(rinf, ctx):
    """An infinity or NaN makes its block (of its head, of keys or values) NaN and leaves the others."""
    rng = np.random.default_rng(8)
    heads, hd, n = 3, 64, 100
    k, v = rows(rng, n, heads, hd), rows(rng, n, heads, hd)
    k[:, 2] *= np.float32(1e37)
    v[40, 1, 5] = np.inf
    k[70, 0, 63] = np.nan
    cache = ctx.kv8(1, heads, hd, 128)
    write(ctx, cache, [k[:90]], [v[:90]], [90])
    for i in range(90, n):
        write(ctx, cache, [k[i:i + 1]], [v[i:i + 1]], [i + 1], single=True)
    check(ctx, cache, [k], [v])
    # the NaN's position once more, with a number
    k[70:, 0] = np.abs(k[69:70, 0])
    write(ctx, cache, [k[70:80]], [v[70:80]], [80])
    got, _ = read(ctx, cache, 0, 64, 16)
    assert np.isfinite(got[:, 1:]).all()
    cache.free()


@pytest.mark.parametrize("layout", ["heads_first", "qkv", "off_by_one", "wide_rows"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strides(rinf, ctx, layout, dtype):
    import torch
    rng = np.random.default_rng(9)
    heads, hd, n = 3, 64, 75
    k, v = rows(rng, n, heads, hd, dtype), rows(rng, n, heads, hd, dtype)
    t = torch.float32 if dtype == "f32" else torch.float16

    def place(shape_only):
        if layout == "heads_first":
            return [torch.full((heads, n, hd), 7.0, dtype=t, device="cuda").permute(1, 0, 2) for _ in range(2)]
        if layout == "qkv":
            buf = torch.full((n, 5 * heads, hd), 7.0, dtype=t, device="cuda")
            return [buf[:, 3 * heads:4 * heads], buf[:, 4 * heads:]]
        if layout == "off_by_one":
            return [torch.full((n * heads * hd + 1,), 7.0, dtype=t, device="cuda")[1:].view(n, heads, hd) for _ in range(2)]
        return [torch.full((n, heads, hd + 9), 7.0, dtype=t, device="cuda")[:, :, :hd] for _ in range(2)]

    dk, dv = place(False)
    dk.copy_(torch.from_numpy(k).cuda())
    dv.copy_(torch.from_numpy(v).cuda())
    cache = ctx.kv8(1, heads, hd, 96)
    lens, starts = i32([n]), i32([0, n])
    torch.cuda.synchronize()
    cache.write_dev(dk, dv, lens, starts)
    ctx.synchronize()
    want = [all_quantised(a.astype(np.float32)).astype(NP[dtype]) for a in (k, v)]
    ok, ov = place(True)
    torch.cuda.synchronize()
    cache.read_dev(0, 1, 0, n, ok, ov)
    ctx.synchronize()
    np.testing.assert_array_equal(ok.cpu().numpy(), want[0])
    np.testing.assert_array_equal(ov.cpu().numpy(), want[1])
    if layout == "qkv":                                  # q's part as it was
        assert bool((ok._base[:, :3 * heads] == 7.0).all())
    cache.free()


def test_read_ranges(rinf, ctx):
    """Any range of any sequences, one output only, and nothing beside it written."""
    import torch
    rng = np.random.default_rng(10)
    heads, hd = 2, 80
    hk = [rows(rng, n, heads, hd) for n in (100, 70, 33)]
    hv = [rows(rng, n, heads, hd) for n in (100, 70, 33)]
    cache = ctx.kv8(3, heads, hd, 100)
    write(ctx, cache, hk, hv, [100, 70, 33])
    full = [all_quantised(np.concatenate([h, np.zeros((100 - len(h), heads, hd), np.float32)])) for h in hk]
    for seq, ns, pos, n in ((0, 1, 0, 1), (0, 2, 31, 2), (1, 1, 5, 60), (0, 3, 0, 33), (0, 1, 63, 37), (2, 1, 100, 0), (3, 0, 0, 9)):
        out = torch.full((ns * n + 2, heads, hd), 7.0, device="cuda")
        torch.cuda.synchronize()
        cache.read_dev(seq, ns, pos, n, out[1:1 + ns * n], None)
        ctx.synchronize()
        got = out.cpu().numpy()
        assert (got[0] == 7.0).all() and (got[-1] == 7.0).all()
        if ns * n:
            np.testing.assert_array_equal(got[1:-1].reshape(ns, n, heads, hd),
                                          np.stack([f[pos:pos + n] for f in full[seq:seq + ns]]))
    cache.free()


def test_batches_that_promise_too_much(rinf, ctx):
    """Starts past the rows or falling, lengths past the cache: what is inside is cached, nothing else is touched."""
    import torch
    rng = np.random.default_rng(11)
    heads, hd = 2, 64
    k, v = rows(rng, 50, heads, hd), rows(rng, 50, heads, hd)
    dk, dv = dev(k), dev(v)
    for starts, lens, hist in (
            ([0, 20, 900], [20, 30], [k[:20], k[20:50]]),              # the second's rows end with the buffer
            ([0, 30, 10], [30, 5], [k[:30], k[:0]]),                   # falling: no rows
            ([0, 0, 50], [0, 70], [k[:0], k[:44]]),                    # positions 20 .. 70 of a cache of 64
            ([0, 50, 50], [40, 9], [k[10:50], k[:0]])):                # rows before position 0
        cache = ctx.kv8(2, heads, hd, 64)
        d_lens, d_starts = i32(lens), i32(starts)
        torch.cuda.synchronize()
        cache.write_dev(dk, dv, d_lens, d_starts)
        ctx.synchronize()
        if lens == [0, 70]:
            got, _ = read(ctx, cache, 1, 20, 44)
            full = np.concatenate([np.zeros((20, heads, hd), np.float32), k[:44]])
            np.testing.assert_array_equal(got, all_quantised(full)[20:])
        else:
            check(ctx, cache, hist, [x if x is None else v[:0] if not len(x) else v[[np.flatnonzero((k == y).all((1, 2)))[0] for y in x]] for x in hist])
        cache.free()


def test_captured_steps(rinf, ctx):
    """One graph of a single-token write, replayed as the device lengths and rows change."""
    import torch
    rng = np.random.default_rng(12)
    heads, hd, seqs = 2, 64, 3
    cache = ctx.kv8(seqs, heads, hd, 128)
    n0 = [30, 0, 61]
    hk = [rows(rng, n, heads, hd) for n in n0]
    hv = [rows(rng, n, heads, hd) for n in n0]
    write(ctx, cache, hk, hv, n0)
    st = torch.cuda.Stream()
    k, v, lens = dev(rows(rng, seqs, heads, hd)), dev(rows(rng, seqs, heads, hd)), i32(n0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        cache.write_dev(k, v, lens, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(6):
        nk, nv = rows(rng, seqs, heads, hd), rows(rng, seqs, heads, hd)
        hk = [np.concatenate([h, x[None]]) for h, x in zip(hk, nk)]
        hv = [np.concatenate([h, x[None]]) for h, x in zip(hv, nv)]
        k.copy_(dev(nk)), v.copy_(dev(nv)), lens.copy_(i32([len(h) for h in hk]))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(ctx, cache, hk, hv)
    cache.free()


def test_refusals(rinf, ctx):
    import ctypes

    import torch
    lib, h = rinf.load_library(), ctypes.c_void_p()
    for args in ((0, 1, 64, 32), (1, 0, 64, 32), (1, 1, 0, 32), (1, 1, 257, 32), (1, 1, 64, 0), (65536, 1, 64, 32),
                 (1, 65536, 64, 32), (1, 1, 64, 1 << 31), (65535, 65535, 256, 1 << 30)):
        assert lib.qg_kv8_create(ctx.h, *args, ctypes.byref(h)) == 7 and not h.value, args
    assert lib.qg_kv8_create(ctx.h, 1, 1, 1, 1, None) == 1
    ctx.fail_allocations(1)
    assert lib.qg_kv8_create(ctx.h, 1, 1, 64, 32, ctypes.byref(h)) == 6 and not h.value
    cache = ctx.kv8(2, 2, 64, 64)
    k = torch.zeros(2, 2, 64, device="cuda")
    lens = i32([1, 1])

    def rows_(**kw):
        d = dict(data=k.data_ptr(), type=0, ld_row=128, ld_head=64)
        d.update(kw)
        return rinf.Rows(**d)

    def call(b=None, rk=None, rv=None):
        b = b or rinf.Batch(2, None, lens.data_ptr())
        return lib.qg_kv8_write_dev(ctx.h, cache.h, ctypes.byref(b), ctypes.byref(rk or rows_()), ctypes.byref(rv or rows_()), None)

    assert call() == 0
    assert call(rk=rows_(type=12)) == 2 and call(rk=rows_(type=1)) == 2          # Q4_K; k f16 and v f32
    assert call(rk=rows_(data=None)) == 1 and call(rv=rows_(data=k.data_ptr() + 2)) == 1
    assert call(rk=rows_(ld_row=1 << 62)) == 7
    assert call(b=rinf.Batch(3, None, lens.data_ptr())) == 7                      # one row per sequence
    assert call(b=rinf.Batch(2, None, None)) == 1 and call(b=rinf.Batch(2, None, lens.data_ptr() + 1)) == 1
    assert call(b=rinf.Batch(1 << 31, lens.data_ptr(), lens.data_ptr())) == 7
    assert call(b=rinf.Batch(1 << 28, lens.data_ptr(), lens.data_ptr())) == 7
    assert lib.qg_kv8_create(ctx.h, 8193, 8192, 1, 1, ctypes.byref(h)) == 7
    assert lib.qg_kv8_write_dev(ctx.h, cache.h, None, None, None, None) == 1
    out = rows_()
    read_ = lambda *a, o=out: lib.qg_kv8_read_dev(ctx.h, cache.h, *a, ctypes.byref(o), None, None)  # noqa: E731
    assert read_(0, 1, 0, 2) == 0
    assert read_(0, 3, 0, 1) == 7 and read_(2, 1, 0, 1) == 7 and read_(0, 1, 64, 1) == 7 and read_(0, 1, 2 ** 64 - 1, 2) == 7
    assert read_(0, 1, 0, 2, o=rows_(ld_row=64)) == 7 and read_(0, 1, 0, 2, o=rows_(ld_head=0)) == 7   # outputs that overlap
    other = rinf.GpuContext(0)
    b = rinf.Batch(2, None, lens.data_ptr())
    assert lib.qg_kv8_write_dev(other.h, cache.h, ctypes.byref(b), ctypes.byref(out), ctypes.byref(out), None) == 1
    assert lib.qg_kv8_free(other.h, cache.h) == 1
    other.close()
    with pytest.raises(rinf.QgemvError):
        cache.write_dev(k, k[:, :1], lens)
    torch.cuda.synchronize()
    handle = cache.h
    cache.free()
    assert lib.qg_kv8_free(ctx.h, handle) == 1
