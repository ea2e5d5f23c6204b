"""The decode-step model on 8-bit caches (qg_model_use_kv8) and its token
probabilities (qg_model_logprobs).

The reference is the forward pass in numpy on the oracle's mat-vecs and norms,
with every layer's keys and values as the cache holds them at each step
(test_kv8_gpu.quantised).  The device's keys and values differ from it by f32
rounding, so a value next to the middle between two codes may take the other
one: one code of a position is 1/127 of its block's largest value at most, times
the weight of that position, and a handful of the tens of thousands of codes here
(their relative distance, 1e-6 of a step's 2^7 codes) can flip.  TOL holds for
a few flips and is a tenth of what the quantisation itself changes."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import normwise_err
from test_decode_gpu import SMALL, build
from test_kv8_gpu import all_quantised

pytestmark = pytest.mark.gpu

TOL = 2e-3


class Forward:
    """transformer.rs:63-98 for one sequence, keys and values through `cached`."""

    def __init__(self, synth, oracle, cfg, mix, seed, cached):
        t = synth.gen_model(cfg, mix, seed)
        self.m, self.v, self.cfg, self.oracle, self.cached = t["mats"], t["vecs"], cfg, oracle, cached
        n = cfg["n_layers"]
        self.hd = cfg["embed_dim"] // cfg["n_heads"]
        self.k, self.val = ([np.zeros((0, cfg["n_kv_heads"], self.hd), np.float32)] * n for _ in range(2))

    def mul(self, slot, l, x):
        raw, dtype, rows, cols = self.m[slot, l]
        return self.oracle.mat_vec_mul(raw, dtype, rows, cols, np.ascontiguousarray(x, np.float32))

    def vec(self, name, l, n):
        return self.v.get((name, l), np.zeros(n, np.float32))

    def rope(self, x, pos):
        i = np.arange(self.hd // 2)
        a = np.float32(pos) * (np.float32(1) / np.power(np.float32(self.cfg["rope_base"]), (2 * i / self.hd).astype(np.float32)))
        c, s, y = np.cos(a), np.sin(a), np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 0::2] * s + x[:, 1::2] * c
        return y.astype(np.float32)

    def chunk(self, tokens, embedding):
        """Tokens that go through a layer together: each sees the cache as it is
        when all of them are written.  The last one's logits."""
        c, hd = self.cfg, self.hd
        h, g = embedding[np.asarray(tokens)].astype(np.float32), c["n_heads"] // c["n_kv_heads"]
        n = len(h)
        for l in range(c["n_layers"]):
            before = len(self.k[l])
            q, k, v = [], [], []
            for i in range(n):
                x = self.oracle.rmsnorm(h[i], self.v["attn_norm", l], c["norm_eps"])
                q.append(self.rope((self.mul("wq", l, x) + self.vec("bq", l, c["embed_dim"])).reshape(-1, hd), before + i))
                k.append(self.rope((self.mul("wk", l, x) + self.vec("bk", l, c["n_kv_heads"] * hd)).reshape(-1, hd), before + i))
                v.append((self.mul("wv", l, x) + self.vec("bv", l, c["n_kv_heads"] * hd)).reshape(-1, hd).astype(np.float32))
            self.k[l], self.val[l] = np.concatenate([self.k[l], np.stack(k)]), np.concatenate([self.val[l], np.stack(v)])
            kq, vq = self.cached(self.k[l]).astype(np.float64), self.cached(self.val[l]).astype(np.float64)
            for i in range(n):
                out = []
                for a in range(c["n_heads"]):
                    s = kq[:before + i + 1, a // g] @ q[i][a].astype(np.float64) / np.sqrt(hd)
                    e = np.exp(s - s.max())
                    out.append(e @ vq[:before + i + 1, a // g] / e.sum())
                y = h[i] + self.mul("wo", l, np.concatenate(out))
                x = self.oracle.rmsnorm(y.astype(np.float32), self.v["ffn_norm", l], c["norm_eps"])
                a, u = self.mul("gate", l, x).astype(np.float64), self.mul("up", l, x)
                h[i] = (y + self.mul("down", l, a / (1 + np.exp(-a)) * u)).astype(np.float32)
        return self.mul("lm_head", 0, self.oracle.rmsnorm(h[-1], self.v["final_norm", 0], c["norm_eps"]))

    def step(self, token, embedding):
        return self.chunk([token], embedding)


def embedding(rinf, oracle, synth, cfg, mix, seed):
    raw, dtype, rows, cols = synth.gen_model(cfg, mix, seed)["mats"]["token_embd", 0]
    eye = np.eye(cols, dtype=np.float32)
    return np.stack([oracle.mat_vec_mul(raw, dtype, rows, cols, eye[i]) for i in range(cols)], 1)


@pytest.mark.parametrize("embed,heads,kv", [(256, 4, 2), (512, 4, 1), (512, 8, 8), (320, 4, 2), (512, 2, 1)])
def test_steps_against_the_definition(rinf, synth, oracle, ctx, embed, heads, kv):
    """40 tokens one by one, the block of 32 closed and the next one opened; heads of 64, 128, 80 and 256."""
    cfg = dict(SMALL, embed_dim=embed, n_heads=heads, n_kv_heads=kv)
    mix = "q8_0"
    dev, _, _ = build(rinf, synth, oracle, ctx, cfg, mix, 41, 64)
    dev.use_kv8(True)
    table = embedding(rinf, oracle, synth, cfg, mix, 41)
    ref, plain = (Forward(synth, oracle, cfg, mix, 41, f) for f in (all_quantised, lambda x: x))
    logits, away = np.zeros(cfg["vocab_size"], np.float32), []
    for pos in range(40):
        tok = (pos * 37 + 5) % cfg["vocab_size"]
        dev.forward(tok, pos, logits)
        want = ref.step(tok, table)
        err = normwise_err(logits, want)
        away.append(normwise_err(plain.step(tok, table), want))
        assert err <= TOL, (pos, err)
    print("quantisation changes the logits by up to %.1e" % max(away))
    dev.close()


@pytest.mark.parametrize("mix,chunks", [("q4_k_m", [20]), ("q4_k_m", [64]), ("q4_k_m", [65]), ("q8_0", [300]),
                                        ("q5_k_m", [640, 460]), ("q8_0", [10, 65, 1, 124])])
def test_prompts_against_the_definition(rinf, synth, oracle, ctx, mix, chunks):
    """The batched prefills: one chunk of up to 64 tokens, one wide chunk, 1100 tokens in two wide ones (one call),
    and calls on top of each other that end inside blocks; steps after them."""
    cfg = dict(SMALL, embed_dim=512, n_heads=4, n_kv_heads=2)
    n = sum(chunks)
    dev, _, _ = build(rinf, synth, oracle, ctx, cfg, mix, 43, n + 8)
    dev.use_kv8(True)
    table = embedding(rinf, oracle, synth, cfg, mix, 43)
    ref = Forward(synth, oracle, cfg, mix, 43, all_quantised)
    prompt = np.arange(n) * 37 % cfg["vocab_size"]
    logits, at = np.zeros(cfg["vocab_size"], np.float32), 0
    if chunks[0] == 640:
        dev.prefill(prompt, logits)
    for m in chunks:
        if chunks[0] != 640:
            dev.prefill(prompt[at:at + m], logits)
        want = ref.chunk(prompt[at:at + m], table)
        at += m
        if chunks[0] != 640 or at == n:
            assert normwise_err(logits, want) <= TOL
    for i in range(3):
        dev.forward(i, n + i, logits)
        assert normwise_err(logits, ref.step(i, table)) <= TOL
    dev.close()


def test_graphs_and_generate(rinf, synth, oracle, ctx):
    """Replayed and launched steps are the same bits, also with eager work between them; generate is its steps."""
    cfg = dict(SMALL)
    dev, _, _ = build(rinf, synth, oracle, ctx, cfg, "q4_k_m", 45, 96)
    dev.use_kv8(True)
    prompt = np.arange(1, 50) % cfg["vocab_size"]
    got = {}
    for graphs in (True, False):
        dev.use_graphs(graphs)
        dev.reset()
        dev.prefill(prompt)
        out = []
        for i in range(20):
            logits = np.zeros(cfg["vocab_size"], np.float32)
            dev.forward(i, 49 + i, logits)
            out.append(logits.tobytes())
        got[graphs] = out
    assert got[True] == got[False]
    dev.use_graphs(True)
    a, _, _ = dev.generate(prompt, 30)
    b, _, _ = dev.generate(prompt, 30)
    recent = list(prompt)
    dev.reset()
    dev.prefill(prompt)
    c = []
    for i in range(30):
        c.append(dev.sample_greedy(recent[-64:]))
        recent.append(c[-1])
        dev.forward(c[-1], 49 + i)
    assert list(a) == list(b) == c
    dev.close()


def test_switching_and_memory(rinf, synth, oracle, ctx):
    """Back to f32 the model gives its old bits; 8-bit caches take a quarter of the memory; a failed switch leaves the model as it was."""
    cfg = dict(SMALL, embed_dim=512, n_heads=4, n_kv_heads=4)
    dev, _, _ = build(rinf, synth, oracle, ctx, cfg, "q8_0", 46, 60000)
    prompt = np.arange(70) % cfg["vocab_size"]
    out = []
    for on in (False, True, False, True):
        if on and len(out) == 1:
            for skip in range(6):                     # layer caches, then the buffers
                ctx.fail_allocations(1, skip)
                with pytest.raises(rinf.QgemvError) as e:
                    dev.use_kv8(True)
                assert e.value.status == 6
                ctx.fail_allocations(0)
        dev.use_kv8(on)
        assert dev.seq_len == 0
        logits = np.zeros(cfg["vocab_size"], np.float32)
        dev.prefill(prompt)
        dev.forward(3, 70, logits)
        out.append((logits.tobytes(), dev.resident_bytes()["total"]))
    assert out[0][0] == out[2][0] and out[1][0] == out[3][0] and out[0][0] != out[1][0]
    f32, q8 = 2 * 2 * 60000 * 512 * 4, out[1][1] - (out[0][1] - 2 * 2 * 60000 * 512 * 4)
    assert q8 < 0.25 * f32 + 120e6 and out[3][1] == out[1][1]         # codes, scales and the workspace
    with pytest.raises(rinf.QgemvError):
        dev.forward(cfg["vocab_size"], 71)
    dev.close()


def test_logprobs(rinf, synth, oracle, ctx):
    cfg = dict(SMALL, vocab_size=5000)
    dev, _, _ = build(rinf, synth, oracle, ctx, cfg, "q8_0", 47, 64)
    logits = np.zeros(5000, np.float32)
    dev.prefill(np.arange(10), logits)
    lp = logits.astype(np.float64) - logits.max()
    lp -= np.log(np.exp(lp).sum())
    tokens = np.concatenate([np.arange(5000), [5000, rinf.TOKEN_NONE]])
    got, ent, ids, top = dev.logprobs(tokens, 20)
    # x - m and the sums in f32: see test_logprobs_gpu
    np.testing.assert_allclose(got[:5000], lp, atol=2.0 ** -16, rtol=2.0 ** -21)
    assert np.isnan(got[5000]) and got[5001] == 0
    assert abs(ent + (np.exp(lp) * lp).sum()) <= 2.0 ** -12
    assert list(ids) == list(np.argsort(-logits, kind="stable")[:20])
    np.testing.assert_array_equal(top, got[ids])
    assert dev.sample_greedy([], 1.0) == ids[0]
    none, ent2, _, _ = dev.logprobs()
    assert len(none) == 0 and ent2 == ent
    lib = rinf.load_library()
    assert lib.qg_model_logprobs(dev.h, None, 1, None, None, 0, None, None) == 1
    assert lib.qg_model_logprobs(dev.h, None, 0, None, None, 65, ids.ctypes.data, top.ctypes.data) == 7
    assert lib.qg_model_logprobs(None, None, 0, None, None, 0, None, None) == 1
    assert lib.qg_model_use_kv8(None, 1) == 1
    dev.close()


def test_memory_comes_back(rinf, synth, oracle):
    """Contexts, caches and 8-bit models built and torn down, some of them by their context."""
    import torch

    def once():
        c = rinf.GpuContext(0)
        kept = c.kv8(4, 4, 128, 5000)
        c.kv8(1, 1, 64, 100).free()
        dev, _, _ = build(rinf, synth, oracle, c, dict(SMALL), "q8_0", 48, 4000)
        dev.use_kv8(True)
        dev.prefill(np.arange(100))
        dev.logprobs([1], 2)
        c.synchronize()
        c.close()
        assert kept.h is not None
        kept.free()

    once()
    torch.cuda.synchronize()
    free0 = torch.cuda.mem_get_info()[0]
    for _ in range(4):
        once()
    torch.cuda.synchronize()
    assert free0 - torch.cuda.mem_get_info()[0] < 16 << 20
