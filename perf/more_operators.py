"""Operators of a token step around and in front of its products, as cases that can be timed.

A served model adds a layer's result to the residual stream and normalises the sum for the next product, attends from the
new tokens of many sequences to keys and values that lie in pages of a cache, and reports the log probabilities of tokens.
A user records a computation with such an operator once, keeps its context and executes it on one set of device
buffers after the other; the caches are the user's own buffers, which the operator extends by the new tokens.

Families and the ranges that `draw` covers:
  norm    1 .. 8192 rows of 64 .. 8192 values, bf16 / fp16 / fp32, results in the same type or 8-bit with scales,
          with or without a residual
  attend  1 .. 64 sequences, 1 .. 8192 new tokens each, up to 32768 cached ones, 1 .. 8 heads of keys with 1 .. 16 heads
          of queries each, heads of 64 .. 256, pages of 1 .. 128 tokens, with or without a window, bf16 / fp16 / fp32
  score   1 .. 8192 rows of 1000 .. 131072 logits, up to 20 alternatives, fp32 / bf16 / fp16
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 128
EPSILON = 1e-6


def listed():
    return [
        # one token between two layers, in front of an 8-bit product: the smallest call
        {"name": "norm_bf16_1x4096_8bit", "family": "norm", "type": "bf16", "m": 1, "k": 4096, "residual": True, "quantize": True},
        # a prompt of no round length, rows of an odd length, result in the type of the stream
        {"name": "norm_fp16_777x2601", "family": "norm", "type": "fp16", "m": 777, "k": 2601, "residual": True, "quantize": False},
        # a long prompt in front of an 8-bit product: bound by memory
        {"name": "norm_bf16_8192x7168_8bit", "family": "norm", "type": "bf16", "m": 8192, "k": 7168, "residual": True, "quantize": True},
        # the next token of a single stream: latency, one row of queries against thousands of keys
        {"name": "attend_bf16_1x4096_h32", "family": "attend", "type": "bf16", "b": 1, "n": 1, "mix": "even", "context": 4096,
         "heads": 8, "group": 4, "d": 128, "page": 16, "window": 0},
        # a decoding batch of sequences of very different lengths: bound by reading the cache
        {"name": "attend_bf16_48x16384_h64", "family": "attend", "type": "bf16", "b": 48, "n": 1, "mix": "even", "context": 16384,
         "heads": 8, "group": 8, "d": 128, "page": 64, "window": 0},
        # a chunk of one prompt beside sequences that decode, heads and pages of other sizes
        {"name": "attend_fp16_17x6000_chunk509_d96", "family": "attend", "type": "fp16", "b": 17, "n": 509, "mix": "one",
         "context": 6000, "heads": 4, "group": 4, "d": 96, "page": 32, "window": 0},
        # short chunks in 32 bits, pages that no tile divides, a window
        {"name": "attend_fp32_3x1000_chunk100_d64", "family": "attend", "type": "fp32", "b": 3, "n": 100, "mix": "ragged",
         "context": 1000, "heads": 4, "group": 2, "d": 64, "page": 20, "window": 700},
        # a long prompt: bound by the matrix cores
        {"name": "attend_bf16_prompt8192_h32", "family": "attend", "type": "bf16", "b": 1, "n": 8192, "mix": "even", "context": 0,
         "heads": 8, "group": 4, "d": 128, "page": 64, "window": 0},
        # the token that was drawn, with its alternatives: the latency of a single stream
        {"name": "score_fp32_1x32000_top20", "family": "score", "type": "fp32", "b": 1, "v": 32000, "top": 20},
        # a batch over a vocabulary of odd size, 16-bit logits (many equal ones)
        {"name": "score_bf16_33x50257_top5", "family": "score", "type": "bf16", "b": 33, "v": 50257, "top": 5},
        # a prompt that is scored: many rows, no alternatives
        {"name": "score_bf16_4001x32000", "family": "score", "type": "bf16", "b": 4001, "v": 32000, "top": 0},
        # a large batch over a large vocabulary
        {"name": "score_fp32_256x128256_top20", "family": "score", "type": "fp32", "b": 256, "v": 128256, "top": 20},
    ]


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, unit):
    """One of the sizes that are usual (multiples of `unit`) or any other one, odd ones too."""
    n = _log(rng, lo, hi)
    return max(unit, n // unit * unit) if rng.random() < 0.6 else n


def _cost(c):
    """(elements of both caches, scores that the plain form holds at a time, products) of an attention case."""
    longest = c["context"] + c["n"]
    hq = c["heads"] * c["group"]
    return (2 * c["b"] * longest * c["heads"] * c["d"], c["b"] * c["n"] * hq * longest, 4 * c["b"] * c["n"] * hq * longest * c["d"])


def draw(rng):
    family = rng.choice(["norm", "attend", "attend", "attend", "score"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if family == "norm":
        k = _size(rng, 64, 8192, 64)
        return {"family": family, "type": kind, "m": _log(rng, 1, min(8192, 8192 * 4096 // k)), "k": k,
                "residual": rng.random() < 0.7, "quantize": rng.random() < 0.5}
    if family == "score":
        v = _log(rng, 1000, 131072)
        return {"family": family, "type": rng.choice(["fp32", "bf16", "fp16"]), "b": _log(rng, 1, min(8192, 256 * 128256 // v)),
                "v": v, "top": rng.choice([0, 1, 5, 20])}
    way = rng.choice(["token", "token", "chunk", "chunk", "prompt"])
    c = {"family": family, "type": kind, "b": _log(rng, 1, {"token": 64, "chunk": 16, "prompt": 4}[way]),
         "n": {"token": 1, "chunk": _log(rng, 2, 512), "prompt": _log(rng, 64, 8192)}[way],
         "mix": {"token": "even", "chunk": rng.choice(["ragged", "one"]), "prompt": rng.choice(["even", "ragged"])}[way],
         "context": {"token": _log(rng, 16, 32768), "chunk": rng.choice([0, _log(rng, 16, 8192)]), "prompt": 0}[way],
         "heads": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 4, 5, 8, 16]), "d": rng.choice([64, 80, 96, 128, 128, 192, 256]),
         "page": rng.choice([1, 16, 16, 20, 32, 64, 128]), "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)])}
    while any(x > y for x, y in zip(_cost(c), (2 * 48 * 16385 * 8 * 128 // 3, 32 * 8192 * 8192, 2 * 32 * 8192 * 8192 * 128))):
        if c["b"] > 1:
            c["b"] = c["b"] * 2 // 3
        else:
            c["n"], c["context"] = max(1, c["n"] * 2 // 3), c["context"] * 2 // 3
    return c


def _lengths(case):
    """(new tokens, cached tokens) of each sequence: the case's own, whatever the inputs' seed."""
    rng = random.Random("%(b)d %(n)d %(mix)s %(context)d" % case)
    new, cached = [], []
    for i in range(case["b"]):
        new.append(case["n"] if case["mix"] == "even" or i == 0 else 1 if case["mix"] == "one" else rng.randint(1, case["n"]))
        cached.append(case["context"] if i == 0 or case["context"] < 2 else _log(rng, max(1, case["context"] // 32), case["context"]))
    return new, cached


# ---------------------------------------------------------------- inputs --
def _blocks(n):
    return -(-n // BLOCK)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")
    kind = _TYPES[case["type"]]
    if case["family"] == "norm":
        m, k = case["m"], case["k"]
        x = normal(m, k)
        x[:, :: 97] *= 20.0                       # a few channels of activations are far larger than the rest
        d = {"x": x.to(kind), "weight": (1 + 0.2 * normal(k)).to(kind)}
        if case["residual"]:
            d["residual"] = (2 * normal(m, k)).to(kind)
        return d
    if case["family"] == "score":
        b, v = case["b"], case["v"]
        logits = normal(b, v, dtype=kind).mul_(3.0)
        logits[:, 17::101] = -math.inf            # words that a grammar rules out
        return {"logits": logits, "tokens": (uniform(b) * v).long().clamp(max=v - 1).to(torch.int32)}
    new, cached = _lengths(case)
    h, d, page = case["heads"], case["d"], case["page"]
    t = sum(new)
    owned = [-(-(n + c) // page) for n, c in zip(new, cached)]
    pages = sum(owned)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu().numpy()    # pages lie as they came free
    table = np.full((case["b"], max(owned)), -1, np.int32)
    ends = np.cumsum([0] + owned)
    for i, n in enumerate(owned):
        table[i, :n] = order[ends[i]:ends[i] + n]
    whole = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    return {"query": normal(t, h * case["group"], d, dtype=kind), "key": normal(t, h, d, dtype=kind), "value": normal(t, h, d, dtype=kind),
            "key_cache": normal(pages, page, h, d, dtype=kind), "value_cache": normal(pages, page, h, d, dtype=kind),
            "page_table": whole(table), "cached": whole(cached), "starts": whole(np.cumsum([0] + new))}


# -------------------------------------------------------- the framework's --
class _Program:
    """A recorded computation and the context that executes it."""

    def __init__(self, case):
        odla = importlib.import_module("heterogeneity-aware-lowering-and-optimization_amd").odla
        kind = {"fp32": np.float32, "fp16": np.float16, "bf16": odla.BFLOAT16}[case["type"]]
        self.b = b = odla.HipBuilder()
        self.session = None
        if case["family"] == "norm":
            m, k = case["m"], case["k"]
            got = b.rms_norm(b.arg("x", (m, k), kind), b.arg("weight", (k,), kind), residual=b.arg("residual", (m, k), kind) if case["residual"] else None,
                             epsilon=EPSILON, dtype=odla.FLOAT8_E4M3 if case["quantize"] else kind)
            names = (["q", "scale"] if case["quantize"] else ["y"]) + (["sum"] if case["residual"] else [])
        elif case["family"] == "score":
            got = b.log_probs(b.arg("logits", (case["b"], case["v"]), kind), b.arg("tokens", (case["b"],), np.int32), top=case["top"])
            names = ["log_prob", "entropy"] + (["top_log_prob", "top_token"] if case["top"] else [])
        else:
            new, cached = _lengths(case)
            h, d, page = case["heads"], case["d"], case["page"]
            owned = [-(-(n + c) // page) for n, c in zip(new, cached)]
            cache = (sum(owned), page, h, d)
            got = [b.paged_attention(b.arg("query", (sum(new), h * case["group"], d), kind), b.arg("key", (sum(new), h, d), kind),
                                     b.arg("value", (sum(new), h, d), kind), b.arg("key_cache", cache, kind), b.arg("value_cache", cache, kind),
                                     b.arg("page_table", (case["b"], max(owned)), np.int32), b.arg("cached", (case["b"],), np.int32),
                                     starts=b.arg("starts", (case["b"] + 1,), np.int32), scale=d ** -0.5, window=case["window"])]
            names = ["y"]
        for n, v in zip(names, got):
            b.output(v, n)
        self.session = b.session()

    def __del__(self):
        if getattr(self, "session", None) is not None:
            self.session.close()
        self.b.destroy()


_last = {}   # the program of the case at hand: one at a time


def _program(case):
    key = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    if key not in _last:
        _last.clear()
        _last[key] = _Program(case)
    return _last[key]


def _results(case, inputs):
    """Buffers for what a call computes."""
    empty = lambda *shape, dtype: torch.empty(shape, device="cuda", dtype=dtype)
    if case["family"] == "norm":
        m, k = case["m"], case["k"]
        d = {"q": empty(m, k, dtype=torch.float8_e4m3fn), "scale": empty(m, _blocks(k), dtype=torch.float32)} if case["quantize"] else {
            "y": torch.empty_like(inputs["x"])}
        if case["residual"]:
            d["sum"] = torch.empty_like(inputs["x"])
        return d
    if case["family"] == "score":
        d = {"log_prob": empty(case["b"], dtype=torch.float32), "entropy": empty(case["b"], dtype=torch.float32)}
        if case["top"]:
            d["top_log_prob"] = empty(case["b"], case["top"], dtype=torch.float32)
            d["top_token"] = empty(case["b"], case["top"], dtype=torch.int32)
        return d
    return {"y": torch.empty_like(inputs["query"])}


class _State:
    def __init__(self, case, inputs):
        self.case, self.inputs = case, inputs
        if own:
            self.program = _program(case)
            results = _results(case, inputs)
            b = self.program.b
            self.args = [(b.args[n][0], t.data_ptr()) for n, t in inputs.items()]
            self.outs = [(b.outs[n][0], t.data_ptr()) for n, t in results.items()]
            self.results = dict(results, **{n: inputs[n] for n in ("key_cache", "value_cache") if n in inputs})


def prepare(case, seed):
    return _State(case, _inputs(case, seed))


def run(state):
    if not own:
        return _PLAIN[state.case["family"]](state.case, state.inputs)
    s = state.program.session
    for h, p in state.args:
        s.L.odla_BindToArgument(h, p, s.ctx)
    for h, p in state.outs:
        s.L.odla_BindToOutput(h, p, s.ctx)
    s.execute()
    return state.results


# ----------------------------------------------------------- plain forms --
def _plain_norm(case, d):
    m, k, kind = case["m"], case["k"], _TYPES[case["type"]]
    x = d["x"].float() + d["residual"].float() if case["residual"] else d["x"].float()
    y = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPSILON) * d["weight"].float()
    if case["quantize"]:
        blocks = torch.nn.functional.pad(y, (0, _blocks(k) * BLOCK - k)).reshape(m, -1, BLOCK)
        scale = torch.clamp(blocks.abs().amax(2) / 448.0, min=2.0 ** -126)
        out = {"q": (blocks / scale[:, :, None]).reshape(m, -1)[:, :k].to(torch.float8_e4m3fn).contiguous(), "scale": scale}
    else:
        out = {"y": y.to(kind)}
    if case["residual"]:
        out["sum"] = x.to(kind)
    return out


def _plain_attend(case, d):
    h, g, dim, page, b = case["heads"], case["group"], case["d"], case["page"], case["b"]
    starts, cached, table = d["starts"].long(), d["cached"].long(), d["page_table"].long()
    count = starts[1:] - starts[:-1]
    token = torch.arange(d["query"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, token, right=True) - 1
    step = token - starts[seq]
    # the new tokens' keys and values join the cache
    at = cached[seq] + step
    slot = table[seq, at // page] * page + at % page
    d["key_cache"].view(-1, h, dim)[slot] = d["key"]
    d["value_cache"].view(-1, h, dim)[slot] = d["value"]
    # every sequence's keys side by side, padded to the longest
    most, longest = case["n"], case["context"] + case["n"]
    place = torch.arange(longest, device="cuda")
    where = table[:, place // page].clamp(min=0) * page + place % page                                     # [b, longest]
    real = place[None, :] < (cached + count)[:, None]
    gathered = lambda cache: torch.where(real[:, :, None, None], cache.view(-1, h, dim)[where].float(), 0.0)
    keys = gathered(d["key_cache"]).permute(0, 2, 3, 1).contiguous()                                      # [b, h, dim, longest]
    values = gathered(d["value_cache"]).permute(0, 2, 1, 3).contiguous()
    queries = torch.zeros((b, most, h, g, dim), device="cuda")
    queries[seq, step] = d["query"].float().reshape(-1, h, g, dim)
    queries = queries.permute(0, 2, 1, 3, 4).reshape(b * h, most * g, dim)
    scores = torch.bmm(queries, keys.reshape(b * h, dim, longest)).mul_(dim ** -0.5).reshape(b, h, most, g, longest)
    last = cached[:, None] + torch.arange(most, device="cuda")                                              # a new token's own place
    seen = place <= last[:, :, None]
    if case["window"]:
        seen &= place > (last - case["window"])[:, :, None]
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores = scores.sub_(scores.amax(4, keepdim=True)).exp_()
    total = scores.sum(4, keepdim=True)
    y = torch.bmm(scores.reshape(b * h, most * g, longest), values.reshape(b * h, longest, dim)).reshape(b, h, most, g, dim) / total
    y = y.permute(0, 2, 1, 3, 4)[seq, step].reshape(-1, h * g, dim)
    return {"y": y.to(d["query"].dtype), "key_cache": d["key_cache"], "value_cache": d["value_cache"]}


def _plain_score(case, d):
    logits = d["logits"].float()
    most = logits.amax(1, keepdim=True)
    w = torch.exp(logits - most)
    total = w.sum(1, keepdim=True)
    norm = most + torch.log(total)
    out = {"log_prob": (logits.gather(1, d["tokens"].long()[:, None]) - norm)[:, 0],
           "entropy": torch.log(total[:, 0]) + (torch.where(w > 0, w * (most - logits), 0.0).sum(1) / total[:, 0])}
    if case["top"]:
        ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)
        out["top_log_prob"] = ranked[:, :case["top"]] - norm
        out["top_token"] = order[:, :case["top"]].to(torch.int32).contiguous()
    return out


_PLAIN = {"norm": _plain_norm, "attend": _plain_attend, "score": _plain_score}


# ------------------------------------------------------------------ work --
def work(case):
    """Inputs and results once each (of the caches the keys and values that some new token attends to, and the new ones
    written), and the operations of the products and of one exponential and the sums for each logit or score."""
    es = _BYTES[case["type"]]
    if case["family"] == "norm":
        m, k = case["m"], case["k"]
        result = m * k + 4 * m * _blocks(k) if case["quantize"] else m * k * es
        return {"bytes": m * k * es * (3 if case["residual"] else 1) + k * es + result, "flops": 6 * m * k}
    if case["family"] == "score":
        return {"bytes": case["b"] * (case["v"] * es + 12 + 8 * case["top"]), "flops": 4 * case["b"] * case["v"]}
    new, cached = _lengths(case)
    hq, window = case["heads"] * case["group"], case["window"]
    reach = lambda p: min(p + 1, window) if window else p + 1               # keys that the token at place p attends to
    scores = sum(reach(c + i) for n, c in zip(new, cached) for i in range(n))
    read = sum(min(c, window - 1) if window else c for c in cached)
    t = sum(new)
    return {"bytes": es * case["d"] * (2 * t * hq + 2 * case["heads"] * (read + 2 * t)), "flops": (4 * case["d"] + 4) * hq * scores}


# ----------------------------------------------------------------- exact --
def _exact_e4m3(x):
    """The e4m3 value nearest to each 64-bit one (ties to even), |x| <= 448."""
    exponent = np.maximum(np.frexp(x)[1] - 1, -6)
    unit = np.ldexp(1.0, exponent - 3)
    return np.rint(x / unit) * unit


def exact(case, seed):
    d = _inputs(case, seed)
    if case["family"] == "norm":
        x = d["x"].double().cpu().numpy()
        if case["residual"]:
            x = x + d["residual"].double().cpu().numpy()
        y = x / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + EPSILON) * d["weight"].double().cpu().numpy()
        out = {"y": y}
        if case["quantize"]:
            scale = np.maximum(np.maximum.reduceat(np.abs(y), np.arange(0, case["k"], BLOCK), axis=1) / 448.0, 2.0 ** -126)
            out = {"q": _exact_e4m3(y / np.repeat(scale, BLOCK, axis=1)[:, :case["k"]]), "scale": scale}
        if case["residual"]:
            out["sum"] = x
        return out
    if case["family"] == "score":
        out = {"log_prob": [], "entropy": [], "top_log_prob": [], "top_token": []}
        tokens = d["tokens"].tolist()
        for r in range(case["b"]):
            l = d["logits"][r].double()
            norm = torch.logsumexp(l, 0)
            p = torch.exp(l - norm)
            out["log_prob"].append(l[tokens[r]] - norm)
            out["entropy"].append(torch.sum(torch.where(p > 0, p * (norm - l), 0.0)))
            if case["top"]:
                order = np.lexsort((np.arange(case["v"]), -l.cpu().numpy()))[:case["top"]]
                out["top_log_prob"].append(l[torch.from_numpy(order.copy()).cuda()] - norm)
                out["top_token"].append(torch.from_numpy(order.astype(np.int32)))
        return {n: torch.stack(v) for n, v in out.items() if v}
    h, g, dim, page = case["heads"], case["group"], case["d"], case["page"]
    new, cached = _lengths(case)
    caches = {n: d[n].double() for n in ("key_cache", "value_cache")}
    lines, first = [], 0
    for i, (n, c) in enumerate(zip(new, cached)):
        slots = [(int(p), o) for p in d["page_table"][i].tolist() for o in range(page)][:c + n]
        p, o = (torch.tensor(v, device="cuda") for v in zip(*slots))
        for name in ("key", "value"):
            caches[name + "_cache"][p[c:], o[c:]] = d[name][first:first + n].double()
        y = torch.empty((n, h * g, dim), dtype=torch.float64, device="cuda")
        place = torch.arange(c + n, device="cuda")
        part = max(1, (1 << 27) // (c + n))      # queries at a time
        for head in range(h):
            k, v = (caches[name][p, o, head] for name in ("key_cache", "value_cache"))
            for q in range(head * g, (head + 1) * g):
                for at in range(0, n, part):
                    to = min(n, at + part)
                    s = d["query"][first + at:first + to, q].double() @ k.t() / math.sqrt(dim)
                    own_place = torch.arange(c + at, c + to, device="cuda")[:, None]
                    hidden = place > own_place
                    if case["window"]:
                        hidden |= place <= own_place - case["window"]
                    y[at:to, q] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
        lines.append(y)
        first += n
    return {"y": torch.cat(lines), **caches}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(24)]:
        w = work(c)
        print("%-190s %10.3f MB %10.3f GFLOP" % (c, w["bytes"] / 1e6, w["flops"] / 1e9))
