"""The 8-bit KV cache, attention over it and token log probabilities, as cases
that can be timed and compared.

* ``write``   keys and values of new tokens into a cache that holds 8-bit codes
              with one scale per 32 positions and head, and the touched
              positions read back;
* ``attend``  attention of new tokens over such a cache: prompts, one token per
              sequence, ragged batches, a sliding window;
* ``score``   log probabilities of given tokens, the entropy and the most
              likely alternatives of rows of logits.

``run`` computes an operator in its plain form in f32 or, with ``own`` set,
calls the package.  ``exact`` is the definition in f64.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import sys

import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parent.parent
PKG_NAME = "rust_inference_amd"
BLOCK = 32                    # positions that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16}
TINY = 2.0 ** -126            # a smaller scale is zero


def _package():
    """rust-inference_amd/ (a hyphenated directory) as rust_inference_amd."""
    if PKG_NAME not in sys.modules:
        d = ROOT / "rust-inference_amd"
        spec = importlib.util.spec_from_file_location(PKG_NAME, d / "__init__.py",
                                                      submodule_search_locations=[str(d)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[PKG_NAME] = mod
        spec.loader.exec_module(mod)
    return sys.modules[PKG_NAME]


_ctx = []


def _context():
    if not _ctx:
        _ctx.append(_package().GpuContext(0))
    return _ctx[0]


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decoded token of the small model of a chat: the smallest write
        {"name": "write_step_0_5b", "kind": "write", "type": "f32", "seqs": 1, "kv_heads": 2, "hd": 64,
         "cached": 48, "rows": 1, "ragged": False},
        # a document as the prompt of an 8B model, an odd number of tokens
        {"name": "write_prompt_8b_1001", "kind": "write", "type": "f32", "seqs": 1, "kv_heads": 8, "hd": 128,
         "cached": 0, "rows": 1001, "ragged": False},
        # prompts of different lengths that a server takes in together
        {"name": "write_prompts_32_f16", "kind": "write", "type": "f16", "seqs": 32, "kv_heads": 8, "hd": 128,
         "cached": 0, "rows": 2048, "ragged": True},
        # a decoded token of the small model early in a chat: the smallest attention
        {"name": "attend_step_0_5b_49", "kind": "attend", "type": "f32", "seqs": 1, "heads": 14, "kv_heads": 2,
         "hd": 64, "cached": 48, "rows": 1, "ragged": False, "window": 0},
        # the same of a 7B model at the end of a long conversation
        {"name": "attend_step_7b_2256", "kind": "attend", "type": "f32", "seqs": 1, "heads": 28, "kv_heads": 4,
         "hd": 128, "cached": 2255, "rows": 1, "ragged": False, "window": 0},
        # a server's decode step: 64 conversations of different lengths
        {"name": "attend_steps_64_f16", "kind": "attend", "type": "f16", "seqs": 64, "heads": 32, "kv_heads": 8,
         "hd": 128, "cached": 8191, "rows": 1, "ragged": True, "window": 0},
        # a decoded token over a whole book
        {"name": "attend_step_131072", "kind": "attend", "type": "f32", "seqs": 1, "heads": 32, "kv_heads": 8,
         "hd": 128, "cached": 131071, "rows": 1, "ragged": False, "window": 0},
        # the document's prompt
        {"name": "attend_prompt_8b_1001", "kind": "attend", "type": "f32", "seqs": 1, "heads": 32, "kv_heads": 8,
         "hd": 128, "cached": 0, "rows": 1001, "ragged": False, "window": 0},
        # the next turns of four conversations, each token over the 4096 before it
        {"name": "attend_turns_4_window_f16", "kind": "attend", "type": "f16", "seqs": 4, "heads": 32, "kv_heads": 8,
         "hd": 128, "cached": 6000, "rows": 2048, "ragged": True, "window": 4096},
        # a decoded token's probability and the eight most likely ones
        {"name": "score_step_152064", "kind": "score", "type": "f32", "rows": 1, "cols": 152064, "given": 1, "k": 8,
         "masked": False},
        # the same for a batch of sequences whose grammar rules tokens out
        {"name": "score_steps_64_top20", "kind": "score", "type": "f32", "rows": 64, "cols": 128256, "given": 1,
         "k": 20, "masked": True},
        # the perplexity of a text
        {"name": "score_text_2048_f16", "kind": "score", "type": "f16", "rows": 2048, "cols": 151936, "given": 1,
         "k": 0, "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _cost(case):
    """Seconds, roughly, on a card of 4 TB/s and 200 TFLOP/s."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 2e14


def _draw(rng):
    kind, t = rng.choice(["write", "attend", "attend", "score"]), rng.choice(["f32", "f16"])
    if kind == "score":
        return {"kind": kind, "type": t, "rows": _log(rng, 1, 2048), "cols": _log(rng, 2000, 152064),
                "given": rng.choice([1, 1, 4]), "k": rng.choice([0, 1, 5, 20, 64]), "masked": rng.random() < 0.3}
    hd = rng.choice([64, 64, 128, 128, 128, 256, 80, 96, 40])
    kv = rng.choice([1, 2, 4, 8])
    step = rng.random() < 0.5
    c = {"kind": kind, "type": t, "seqs": _log(rng, 1, 128 if step else 16), "kv_heads": kv, "hd": hd,
         "cached": _log(rng, 1, 60000 if kind == "attend" else 2000) if step or rng.random() < 0.5 else 0,
         "rows": 1 if step else _log(rng, 2, 3000), "ragged": rng.random() < 0.5}
    if kind == "write":
        return c
    return dict(c, heads=kv * rng.choice([1, 2, 4, 7, 8]), window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if c["kind"] == "attend" and (c["seqs"] * (c["cached"] + c["rows"]) * c["kv_heads"] * c["hd"] > 1.5e8 or
                                      c["seqs"] * c["heads"] * c["rows"] * (c["cached"] + c["rows"]) > 2.2e9):
            continue          # the plain form's score matrix and f32 cache
        if _cost(c) <= most:
            return c


# ------------------------------------------------------------------- batches

def _batch(case):
    """(tokens cached before the call, tokens of the call) of every sequence.
    Ragged: spread over the range by two irrational steps, the first one full.
    Writes start at the same position everywhere (one range is read back)."""
    old, new = [], []
    for i in range(case["seqs"]):
        u, w = (i * 0.6180339887498949) % 1, (i * 0.7548776662466927) % 1
        full = not case["ragged"] or i == 0
        old.append(case["cached"] if full or case["kind"] == "write" else int(case["cached"] * u))
        new.append(case["rows"] if full else max(1, int(case["rows"] * w)))
    return old, new


def _index(old, new):
    """Sequence and place within its sequence of every row of the batch."""
    n = torch.tensor(new, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), n)
    place = torch.arange(int(sum(new)), device="cuda") - (torch.cumsum(n, 0) - n)[seq]
    return seq, place


def _device_batch(old, new):
    """The batch as the package takes it: cached positions after the call, and
    the rows' starts (None: one row per sequence)."""
    lens = torch.tensor([a + b for a, b in zip(old, new)], dtype=torch.int32, device="cuda")
    if all(b == 1 for b in new):
        return lens, None
    starts = [0]
    for b in new:
        starts.append(starts[-1] + b)
    return lens, torch.tensor(starts, dtype=torch.int32, device="cuda")


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _channels(case, gen):
    """Keys differ in size from channel to channel, a few of them by much."""
    c = torch.exp(0.5 * torch.randn(case["kv_heads"], case["hd"], generator=gen, device="cuda"))
    return c / c.square().mean(-1, keepdim=True).sqrt()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------- prepare

def _inputs(case, seed):
    """The seeded tensors of a case."""
    gen = _gen(seed)
    if case["kind"] == "score":
        rows, cols = case["rows"], case["cols"]
        x = torch.randn(rows, cols, generator=gen, device="cuda") * 2.5
        first = torch.randint(0, cols, (rows, case["given"]), generator=gen, device="cuda")
        x.scatter_add_(1, first[:, :1], 12 * torch.rand(rows, 1, generator=gen, device="cuda"))
        if case["masked"]:
            x[:, torch.rand(cols, generator=gen, device="cuda") < 0.1] = -math.inf
        return {"x": x.to(TYPES[case["type"]]), "tokens": first.to(torch.int32)}
    t, heads, hd = TYPES[case["type"]], case["kv_heads"], case["hd"]
    old, new = _batch(case)
    size = _channels(case, gen)
    if case["kind"] == "write":
        n = sum(new)
        o = case["cached"] % BLOCK
        return {"k": (torch.randn(n, heads, hd, generator=gen, device="cuda") * size).to(t),
                "v": _randn((n, heads, hd), gen, t),
                "open_k": (torch.randn(case["seqs"], o, heads, hd, generator=gen, device="cuda") * size).to(t),
                "open_v": _randn((case["seqs"], o, heads, hd), gen, t)}
    L = max(a + b for a, b in zip(old, new))
    return {"q": _randn((sum(new), case["heads"], hd), gen, t) * 1.25,
            "k": (torch.randn(case["seqs"], L, heads, hd, generator=gen, device="cuda") * size).to(t),
            "v": _randn((case["seqs"], L, heads, hd), gen, t)}


def _quantise(x):
    """Codes and scales of f32 [seqs, blocks, 32, heads, hd].  The quotients in
    f64: in f32 one next to a half goes to the other side now and then."""
    s = (x.abs().amax(dim=(2, 4), keepdim=True).double() / 127).float()
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    return torch.round(x.double() / torch.where(s == 0, torch.ones_like(s), s)).to(torch.int8), s


def _blocks(x):
    """[seqs, positions, ...] as blocks, zeros behind the last position."""
    pad = -x.shape[1] % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros((x.shape[0], pad) + tuple(x.shape[2:]))], 1)
    return x.reshape((x.shape[0], -1, BLOCK) + tuple(x.shape[2:]))


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": dict(case)}
    if case["kind"] == "score":
        rows, k = case["rows"], case["k"]
        state.update(d)
        if own:
            f = lambda n, t=torch.float32: torch.zeros(rows, n, dtype=t, device="cuda")  # noqa: E731
            state.update(ctx=_context(), logprob=f(case["given"]), entropy=f(1), top_ids=f(k, torch.int32),
                         top_logprobs=f(k))
            state["work"] = torch.zeros(max(16, _context().logprobs_work(rows, case["cols"], k)), dtype=torch.uint8,
                                        device="cuda")
        torch.cuda.synchronize()
        return state
    old, new = _batch(case)
    state["old"], state["new"] = old, new
    state["seq"], state["place"] = _index(old, new)
    state["lens"], state["starts"] = _device_batch(old, new)
    n = max(new)
    if case["kind"] == "write":
        o = case["cached"] % BLOCK
        state.update(d)
        if own:
            cache = _context().kv8(case["seqs"], case["kv_heads"], case["hd"], case["cached"] + n)
            if o:                                  # the tokens of the block that is open when the call comes
                shape = (case["seqs"] * o, case["kv_heads"], case["hd"])
                lens = torch.full((case["seqs"],), case["cached"], dtype=torch.int32, device="cuda")
                starts = torch.arange(case["seqs"] + 1, dtype=torch.int32, device="cuda") * o
                torch.cuda.synchronize()
                cache.write_dev(d["open_k"].reshape(shape), d["open_v"].reshape(shape), lens, starts)
                _context().synchronize()
            shape = (case["seqs"] * (o + n), case["kv_heads"], case["hd"])
            state.update(cache=cache, out_k=torch.zeros(shape, dtype=d["k"].dtype, device="cuda"),
                         out_v=torch.zeros(shape, dtype=d["k"].dtype, device="cuda"))
    else:
        state["q"] = d["q"]
        if own:
            L = d["k"].shape[1]
            cache = _context().kv8(case["seqs"], case["kv_heads"], case["hd"], L)
            # every sequence's tokens so far, those of the call among them
            starts = torch.arange(case["seqs"] + 1, dtype=torch.int32, device="cuda") * L
            shape = (case["seqs"] * L, case["kv_heads"], case["hd"])
            torch.cuda.synchronize()
            if all(a + b == L for a, b in zip(old, new)):
                cache.write_dev(d["k"].reshape(shape), d["v"].reshape(shape), state["lens"], starts)
            else:
                keep = torch.arange(L, device="cuda")[None] < state["lens"][:, None]
                starts = torch.cat([starts[:1], torch.cumsum(state["lens"], 0).to(torch.int32)])
                k, v = d["k"][keep], d["v"][keep]
                torch.cuda.synchronize()
                cache.write_dev(k, v, state["lens"], starts)
            _context().synchronize()
            state.update(cache=cache, out=torch.zeros_like(d["q"]),
                         work=torch.zeros(max(16, cache.attention_work(d["q"].shape[0], case["heads"])),
                                          dtype=torch.uint8, device="cuda"))
        else:
            inside = torch.arange(d["k"].shape[1], device="cuda")[None] < state["lens"][:, None]
            state["codes"] = [_quantise(_blocks(x.float() * inside[:, :, None, None])) for x in (d.pop("k"), d.pop("v"))]
    torch.cuda.synchronize()
    return state


# ----------------------------------------------------------------------- run

def _run_own(state):
    case = state["case"]
    if case["kind"] == "score":
        k = case["k"]
        state["ctx"].logprobs_dev(state["x"], state["tokens"], state["logprob"], state["entropy"],
                                  state["top_ids"] if k else None, state["top_logprobs"] if k else None,
                                  state["work"])
        out = {"logprob": state["logprob"], "entropy": state["entropy"]}
        return dict(out, ids=state["top_ids"], alternatives=state["top_logprobs"]) if k else out
    if case["kind"] == "write":
        o, n = case["cached"] % BLOCK, max(state["new"])
        state["cache"].write_dev(state["k"], state["v"], state["lens"], state["starts"])
        state["cache"].read_dev(0, case["seqs"], case["cached"] - o, o + n, state["out_k"], state["out_v"])
        return [state["out_k"], state["out_v"]]
    state["cache"].attention_dev(state["q"], state["out"], state["lens"], state["work"], state["starts"],
                                 window=case["window"])
    return state["out"]


def _plain_write(state):
    case = state["case"]
    o, n = case["cached"] % BLOCK, max(state["new"])
    out = []
    for x, before in ((state["k"], state["open_k"]), (state["v"], state["open_v"])):
        y = torch.zeros((case["seqs"], o + n) + tuple(x.shape[1:]), device="cuda")
        y[:, :o] = before.float()
        y[state["seq"], o + state["place"]] = x.float()
        y = _blocks(y)
        codes, s = _quantise(y)
        out.append((codes.float() * s).flatten(1, 2)[:, :o + n].flatten(0, 1).to(x.dtype))
    return out


def _plain_attend(state):
    case = state["case"]
    heads, kv, hd = case["heads"], case["kv_heads"], case["hd"]
    g, n = heads // kv, max(state["new"])
    k, v = ((c.float() * s).flatten(1, 2) for c, s in state["codes"])          # [seqs, L, kv, hd]
    q = torch.zeros(case["seqs"], n, heads, hd, device="cuda")
    q[state["seq"], state["place"]] = state["q"].float()
    q = q.reshape(-1, n, kv, g, hd).permute(0, 2, 3, 1, 4).reshape(-1, kv, g * n, hd)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1 / math.sqrt(hd))
    s = s.reshape(-1, kv, g, n, k.shape[1])
    first = torch.tensor(state["old"], device="cuda")
    p = first[:, None] + torch.arange(n, device="cuda")[None]                   # position of every row
    j = torch.arange(k.shape[1], device="cuda")
    seen = j <= p[..., None]
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(-1, kv, g * n, k.shape[1]), v.permute(0, 2, 1, 3).contiguous())
    o = o.reshape(-1, kv, g, n, hd).permute(0, 3, 1, 2, 4).reshape(-1, n, heads, hd)
    return o[state["seq"], state["place"]].to(state["q"].dtype)


def _plain_score(state):
    x, k = state["x"].float(), state["case"]["k"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    z = e.sum(-1, keepdim=True)
    lp = d - z.log()
    ent = z.log() - torch.where(e > 0, d * e, torch.zeros_like(e)).sum(-1, keepdim=True) / z
    out = {"logprob": lp.gather(1, state["tokens"].long()), "entropy": ent}
    if k:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
        out.update(ids=ids.to(torch.int32), alternatives=lp.gather(1, ids))
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "attend": _plain_attend, "score": _plain_score}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- exact

def _exact_values(x, count):
    """What 8-bit blocks make of the first `count` of x [positions, heads, hd]: f64."""
    x = x.double()[:count]
    out = torch.zeros_like(x)
    for b in range(0, count, BLOCK):
        y = x[b:b + BLOCK]
        s = (y.abs().amax(dim=(0, 2), keepdim=True) / 127).float().double()        # a scale is an f32
        out[b:b + BLOCK] = torch.where(s >= TINY, torch.round(y / s) * s, torch.zeros_like(y))
    return out


def _exact_write(case, d):
    old, new = _batch(case)
    o, n = case["cached"] % BLOCK, max(new)
    out = []
    for x, before in ((d["k"], d["open_k"]), (d["v"], d["open_v"])):
        y, at = torch.zeros((case["seqs"], o + n) + tuple(x.shape[1:]), dtype=torch.float64, device="cuda"), 0
        for i, m in enumerate(new):
            y[i, :o + m] = _exact_values(torch.cat([before[i], x[at:at + m]]), o + m)
            at += m
        out.append(y.flatten(0, 1))
    return out


def _exact_attend(case, d):
    old, new = _batch(case)
    g, at, out = case["heads"] // case["kv_heads"], 0, []
    for i, (a, m) in enumerate(zip(old, new)):
        k, v = _exact_values(d["k"][i], a + m), _exact_values(d["v"][i], a + m)
        rows = torch.zeros(m, case["heads"], case["hd"], dtype=torch.float64, device="cuda")
        for r in range(0, m, 256):
            hi = min(m, r + 256)
            p = torch.arange(a + r, a + hi, device="cuda")[:, None]
            j = torch.arange(a + hi, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden |= p - j >= case["window"]
            for h in range(case["kv_heads"]):
                q = d["q"][at + r:at + hi, h * g:(h + 1) * g].double().transpose(0, 1)
                s = torch.matmul(q, k[:a + hi, h].t().contiguous()) / math.sqrt(case["hd"])
                s = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                rows[r:hi, h * g:(h + 1) * g] = torch.matmul(s, v[:a + hi, h].contiguous()).transpose(0, 1)
        out.append(rows)
        at += m
    return torch.cat(out)


def exact(case, seed):
    if case["kind"] != "score" and case["seqs"] * (case["cached"] + case["rows"]) / BLOCK > 40000:
        return None                                # the blocks are gone through one by one
    d = _inputs(case, seed)
    if case["kind"] == "write":
        return _exact_write(case, d)
    if case["kind"] == "attend":
        return _exact_attend(case, d)
    parts = []
    for x, t in zip(d["x"].split(256), d["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), -1)
        p = lp.exp()
        part = [lp.gather(1, t.long()), -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1, keepdim=True)]
        if case["k"]:
            ids = torch.argsort(x.double(), dim=-1, descending=True, stable=True)[:, :case["k"]]
            part += [ids.to(torch.int32), lp.gather(1, ids)]
        parts.append(part)
    names = ["logprob", "entropy", "ids", "alternatives"]
    return {n: torch.cat([p[i] for p in parts]) for i, n in enumerate(names[:len(parts[0])])}


# --------------------------------------------------------------------- work

def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "score":
        rows, cols, k, g = (case[n] for n in ("rows", "cols", "k", "given"))
        return {"bytes": rows * (cols * size + 8 * k + 8 * g + 4), "flops": 6 * rows * cols}
    old, new = _batch(case)
    row = case["kv_heads"] * case["hd"]
    if case["kind"] == "write":
        o, n = case["cached"] % BLOCK, max(new)
        blocks = case["seqs"] * -(-(o + n) // BLOCK) * case["kv_heads"]
        # new rows in, codes out, codes and scales in, values out; keys and values
        return {"bytes": 2 * (sum(new) * row * (size + 1) + 8 * blocks + case["seqs"] * (o + n) * row * (1 + size)),
                "flops": 2 * 3 * row * (sum(new) + case["seqs"] * (o + n))}
    w, cells, seen = case["window"], 0, 0
    for a, m in zip(old, new):
        lo = max(0, a - w + 1) if w else 0
        cells += a + m - lo
        # sum over the rows' positions p = a .. a + m - 1 of min(p + 1, window)
        full = lambda t: t * (t + 1) // 2  # noqa: E731
        seen += full(a + m) - full(a)
        if w:
            over = lambda t: full(max(0, t - w))  # noqa: E731
            seen -= over(a + m) - over(a)
    q = sum(new) * case["heads"] * case["hd"] * size
    return {"bytes": 2 * q + 2 * cells * row * (1 + 4 / (BLOCK * case["hd"])), "flops": 4 * case["hd"] * case["heads"] * seen}
