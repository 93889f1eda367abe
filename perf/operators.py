"""Operators of a token step behind its attention, as cases that can be timed.

A served model quantises activations to 8-bit floating point in blocks of 128, multiplies them
with weights held the same way, sends tokens through a few of many experts, and draws the next
token from the logits.  A user records a computation with such an operator once, keeps its context
and executes it on one set of device buffers after the other.

Families and the ranges that `draw` covers:
  quantize  1 .. 8192 rows of 64 .. 8192 values, bf16 / fp16 / fp32, whole blocks or not
  gemm      1 .. 8192 rows, 128 .. 8192 columns, 128 .. 8192 terms, results in bf16 / fp16 / fp32
  moe       1 .. 64 tokens, 8 .. 256 experts, 1 .. 8 of them chosen, bf16 / fp16 / fp32 / 8-bit weights
  sample    1 .. 256 rows of 1000 .. 131072 logits, fp32 / bf16 / fp16
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "fp8": 1}
BLOCK = 128


def listed():
    return [
        # the activations of one token in front of a product: the smallest call
        {"name": "quantize_bf16_1x4096", "family": "quantize", "type": "bf16", "m": 1, "k": 4096},
        # the activations of a long prompt
        {"name": "quantize_bf16_8192x7168", "family": "quantize", "type": "bf16", "m": 8192, "k": 7168},
        # one token through a square projection: all weights for one row
        {"name": "gemm_bf16_1x4096x4096", "family": "gemm", "type": "bf16", "m": 1, "n": 4096, "k": 4096},
        # a decoding batch
        {"name": "gemm_bf16_48x7168x2048", "family": "gemm", "type": "bf16", "m": 48, "n": 7168, "k": 2048},
        # a prompt of no round length, rows and terms that end inside a block
        {"name": "gemm_fp16_509x2500x1400", "family": "gemm", "type": "fp16", "m": 509, "n": 2500, "k": 1400},
        # a long prompt: bound by the matrix cores
        {"name": "gemm_bf16_8192x8192x4096", "family": "gemm", "type": "bf16", "m": 8192, "n": 8192, "k": 4096},
        # one token of a decoding step through 8 of 64 experts
        {"name": "moe_bf16_t1_e64k8", "family": "moe", "type": "bf16", "t": 1, "e": 64, "top": 8, "h": 2048, "i": 1024},
        # a decoding batch, which reaches nearly all experts
        {"name": "moe_bf16_t32_e64k8", "family": "moe", "type": "bf16", "t": 32, "e": 64, "top": 8, "h": 2048, "i": 1024},
        # many small experts with 8-bit weights, sizes that no tile divides
        {"name": "moe_fp8_t7_e128k6", "family": "moe", "type": "fp8", "t": 7, "e": 128, "top": 6, "h": 2600, "i": 712},
        # one row of logits: the latency of a single stream
        {"name": "sample_fp32_1x32000", "family": "sample", "type": "fp32", "b": 1, "v": 32000},
        # a batch over a vocabulary of odd size, 16-bit logits (many equal ones)
        {"name": "sample_bf16_33x50257", "family": "sample", "type": "bf16", "b": 33, "v": 50257},
        # a large batch over a large vocabulary
        {"name": "sample_fp32_256x128256", "family": "sample", "type": "fp32", "b": 256, "v": 128256},
    ]


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, unit):
    """One of the sizes that are usual (multiples of `unit`) or any other one, odd ones too."""
    n = _log(rng, lo, hi)
    return max(unit, n // unit * unit) if rng.random() < 0.6 else n


def draw(rng):
    family = rng.choice(["quantize", "gemm", "gemm", "moe", "moe", "sample"])
    if family == "quantize":
        k = _size(rng, 64, 8192, 64)
        return {"family": family, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "m": _log(rng, 1, min(8192, 8192 * 4096 // k)), "k": k}
    if family == "gemm":
        n, k = _size(rng, 128, 8192, 128), _size(rng, 128, 8192, 128)
        return {"family": family, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "m": _log(rng, 1, max(1, min(8192, 8192 * 8192 * 4096 // (2 * n * k)))), "n": n, "k": k}
    if family == "moe":
        kind = rng.choice(["bf16", "bf16", "fp16", "fp8", "fp8", "fp32"])
        e = _log(rng, 8, 256)
        h, i = _size(rng, 128, 4096, 128), _size(rng, 64, 2048, 64)
        while e * h * i > 64 * 2048 * 1024 // (2 if kind == "fp32" else 1):
            e = max(8, e // 2)
            h = max(128, h * 3 // 4)
        return {"family": family, "type": kind, "t": _log(rng, 1, 64), "e": e, "top": rng.randint(1, min(8, e)), "h": h, "i": i}
    v = _log(rng, 1000, 131072)
    return {"family": family, "type": rng.choice(["fp32", "bf16", "fp16"]),
            "b": _log(rng, 1, max(1, min(256, 256 * 128256 // v))), "v": v}


# ---------------------------------------------------------------- inputs --
def _blocks(n):
    return -(-n // BLOCK)


def _padded(x, *sizes):
    """`x` with zeros behind its last dimensions, up to `sizes`."""
    y = x.new_zeros(x.shape[:x.dim() - len(sizes)] + tuple(sizes))
    y[tuple([Ellipsis] + [slice(0, n) for n in x.shape[x.dim() - len(sizes):]])] = x
    return y


def _quantized_rows(x):
    """e4m3 values and a scale for each block of 128 of a row."""
    m, k = x.shape
    blocks = _padded(x.float(), _blocks(k) * BLOCK).reshape(m, -1, BLOCK)
    scale = torch.clamp(blocks.abs().amax(2) / 448.0, min=2.0 ** -126)
    q = (blocks / scale[:, :, None]).reshape(m, -1)[:, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scale


def _quantized_squares(w):
    """e4m3 values and a scale for each block of 128 x 128 of the last two dimensions."""
    r, k = w.shape[-2:]
    rb, kb = _blocks(r), _blocks(k)
    blocks = _padded(w.float(), rb * BLOCK, kb * BLOCK).reshape(-1, rb, BLOCK, kb, BLOCK)
    scale = torch.clamp(blocks.abs().amax((2, 4)) / 448.0, min=2.0 ** -126)
    q = (blocks / scale[:, :, None, :, None]).reshape(w.shape[:-2] + (rb * BLOCK, kb * BLOCK))[..., :r, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), scale.reshape(w.shape[:-2] + (rb, kb))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")
    kind = _TYPES[case["type"]]
    if case["family"] == "quantize":
        x = normal(case["m"], case["k"])
        x[:, :: 97] *= 20.0                       # a few channels of activations are far larger than the rest
        return {"x": x.to(kind)}
    if case["family"] == "gemm":
        a, sa = _quantized_rows(normal(case["m"], case["k"]))
        b, sb = _quantized_squares(normal(case["n"], case["k"]) * 0.02)
        return {"a": a, "sa": sa, "b": b, "sb": sb}
    if case["family"] == "moe":
        t, e, h, i = case["t"], case["e"], case["h"], case["i"]
        dense = torch.bfloat16 if case["type"] == "fp8" else kind
        d = {"x": normal(t, h).to(dense), "router": (normal(e, h) * h ** -0.5).to(dense)}
        if case["type"] == "fp8":
            d["gate_up"], d["gate_up_scale"] = _quantized_squares(normal(e, 2 * i, h, dtype=torch.bfloat16) * h ** -0.5)
            d["down"], d["down_scale"] = _quantized_squares(normal(e, h, i, dtype=torch.bfloat16) * i ** -0.5)
        else:
            d["gate_up"] = normal(e, 2 * i, h, dtype=kind).mul_(h ** -0.5)
            d["down"] = normal(e, h, i, dtype=kind).mul_(i ** -0.5)
        return d
    b, v = case["b"], case["v"]
    logits = (normal(b, v) * 3.0).to(kind)
    logits[uniform(b, v) < 0.01] = -math.inf      # words that a grammar rules out
    pick = lambda *values: torch.tensor(values, device="cuda")[(uniform(b) * len(values)).long().clamp(max=len(values) - 1)]
    return {"logits": logits, "temperature": torch.where(uniform(b) < 0.1, 0.0, 0.3 + uniform(b)),
            "top_k": pick(0, 20, 50, 1000).to(torch.int32), "top_p": pick(0.8, 0.9, 0.95, 1.0).float(),
            "min_p": pick(0.0, 0.0, 0.02, 0.1).float(), "uniform": uniform(b)}


# -------------------------------------------------------- the framework's --
class _Program:
    """A recorded computation and the context that executes it."""

    def __init__(self, case):
        odla = importlib.import_module("heterogeneity-aware-lowering-and-optimization_amd").odla
        types = {"fp32": np.float32, "fp16": np.float16, "bf16": odla.BFLOAT16, "fp8": odla.FLOAT8_E4M3}
        kind = types[case["type"]]
        self.b = b = odla.HipBuilder()
        self.session = None
        if case["family"] == "quantize":
            q, s = b.block_quantize(b.arg("x", (case["m"], case["k"]), kind), names=("q", "scale"))
            b.output(q, "q")
            b.output(s, "scale")
        elif case["family"] == "gemm":
            m, n, k = case["m"], case["n"], case["k"]
            b.output(b.block_gemm(b.arg("a", (m, k), odla.FLOAT8_E4M3), b.arg("sa", (m, _blocks(k))),
                                  b.arg("b", (n, k), odla.FLOAT8_E4M3), b.arg("sb", (_blocks(n), _blocks(k))), kind, name="y"), "y")
        elif case["family"] == "moe":
            t, e, h, i = case["t"], case["e"], case["h"], case["i"]
            dense = odla.BFLOAT16 if case["type"] == "fp8" else kind
            x, router = b.arg("x", (t, h), dense), b.arg("router", (e, h), dense)
            gate_up, down = b.arg("gate_up", (e, 2 * i, h), kind), b.arg("down", (e, h, i), kind)
            scales = {}
            if case["type"] == "fp8":
                scales = {"gate_up_scale": b.arg("gate_up_scale", (e, _blocks(2 * i), _blocks(h))),
                          "down_scale": b.arg("down_scale", (e, _blocks(h), _blocks(i)))}
            b.output(b.mixture_of_experts(x, router, gate_up, down, case["top"], renormalize=True, name="y", **scales), "y")
        else:
            rows = {n: b.arg(n, (case["b"],), np.int32 if n == "top_k" else np.float32)
                    for n in ("temperature", "top_k", "top_p", "min_p", "uniform")}
            b.output(b.sample(b.arg("logits", (case["b"], case["v"]), kind), name="token", **rows), "token")
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


def _results(case):
    """Buffers for what a call computes."""
    empty = lambda *shape, dtype: torch.empty(shape, device="cuda", dtype=dtype)
    if case["family"] == "quantize":
        return {"q": empty(case["m"], case["k"], dtype=torch.float8_e4m3fn),
                "scale": empty(case["m"], _blocks(case["k"]), dtype=torch.float32)}
    if case["family"] == "gemm":
        return {"y": empty(case["m"], case["n"], dtype=_TYPES[case["type"]])}
    if case["family"] == "moe":
        return {"y": empty(case["t"], case["h"], dtype=torch.bfloat16 if case["type"] == "fp8" else _TYPES[case["type"]])}
    return {"token": empty(case["b"], dtype=torch.int32)}


class _State:
    def __init__(self, case, inputs):
        self.case, self.inputs = case, inputs
        if own:
            self.program = _program(case)
            self.results = _results(case)
            b = self.program.b
            self.args = [(b.args[n][0], t.data_ptr()) for n, t in inputs.items()]
            self.outs = [(b.outs[n][0], t.data_ptr()) for n, t in self.results.items()]


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
def _plain_quantize(case, d):
    q, scale = _quantized_rows(d["x"])
    return {"q": q, "scale": scale}


def _values_of_rows(q, scale):
    m, k = q.shape
    return (_padded(q.float(), scale.shape[1] * BLOCK).reshape(m, -1, BLOCK) * scale[:, :, None]).reshape(m, -1)[:, :k]


def _values_of_squares(q, scale):
    r, k = q.shape[-2:]
    spread = scale.repeat_interleave(BLOCK, -2)[..., :r, :].repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * spread


def _plain_gemm(case, d):
    y = _values_of_rows(d["a"], d["sa"]) @ _values_of_squares(d["b"], d["sb"]).t()
    return {"y": y.to(_TYPES[case["type"]])}


def _plain_moe(case, d):
    t, e, top, i = case["t"], case["e"], case["top"], case["i"]
    x = d["x"].float()
    # (64 bits: which experts a token takes must not hang on the order of a sum)
    logits = x.double() @ d["router"].double().t()
    order = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
    weight = torch.exp(logits - logits.amax(1, keepdim=True)).gather(1, order)
    weight = (weight / weight.sum(1, keepdim=True)).float()
    if t * top < e:                              # few tokens: their experts alone, each for its token
        ids = order.reshape(-1)
        part = lambda name: _values_of_squares(d[name][ids], d[name + "_scale"][ids]) if case["type"] == "fp8" else d[name][ids].float()
        both = torch.bmm(part("gate_up"), x.repeat_interleave(top, 0)[:, :, None])[:, :, 0]
        hidden = both[:, :i] * torch.sigmoid(both[:, :i]) * both[:, i:]
        each = torch.bmm(part("down"), hidden[:, :, None])[:, :, 0].reshape(t, top, -1)
        y = (each * weight[:, :, None]).sum(1)
    else:                                        # many: every expert for every token, the weight of the others is zero
        whole = lambda name: _values_of_squares(d[name], d[name + "_scale"]) if case["type"] == "fp8" else d[name].float()
        both = (x @ whole("gate_up").reshape(e * 2 * i, -1).t()).reshape(t, e, 2 * i)
        hidden = both[:, :, :i] * torch.sigmoid(both[:, :, :i]) * both[:, :, i:]
        share = x.new_zeros(t, e).scatter_(1, order, weight)
        hidden = (hidden * share[:, :, None]).transpose(0, 1).contiguous()
        y = torch.bmm(hidden, whole("down").transpose(1, 2).contiguous()).sum(0)
    return {"y": y.to(d["x"].dtype)}


def _plain_sample(case, d):
    # (64 bits: a token is a whole number, and whether a sum passes a border decides it)
    v = case["v"]
    logits = d["logits"].double()
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    most = logits.amax(1, keepdim=True)
    temperature = d["temperature"].double()[:, None]
    w = torch.where(logits == most, 1.0, torch.exp((logits - most) / torch.where(temperature > 0, temperature, 1.0)))
    w = torch.where(logits == -math.inf, 0.0, w)
    ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)
    place = torch.arange(v, device=w.device)[None, :]
    top_k = d["top_k"].long()[:, None]
    top_k = torch.where((top_k <= 0) | (top_k > v), v, top_k)
    top_k = torch.where(temperature > 0, top_k, 1)
    ws = torch.where(place < top_k, w.gather(1, order), 0.0)
    before = ws.cumsum(1) - ws
    top_p, min_p = d["top_p"].double()[:, None], d["min_p"].double()[:, None]
    kept = (place < top_k) & ((top_p >= 1) | (before < top_p * ws.sum(1, keepdim=True)) | (place == 0)) & ((ws >= min_p) | (place == 0))
    w = torch.where(torch.zeros_like(kept).scatter_(1, order, kept), w, 0.0)
    sums = w.cumsum(1)
    target = d["uniform"].double()[:, None] * sums[:, -1:]
    token = (sums <= target).sum(1, keepdim=True)
    last = torch.where(w > 0, place, -1).amax(1, keepdim=True)
    return {"token": torch.minimum(token, last)[:, 0].to(torch.int32)}


_PLAIN = {"quantize": _plain_quantize, "gemm": _plain_gemm, "moe": _plain_moe, "sample": _plain_sample}


# ------------------------------------------------------------------ work --
def work(case):
    """Inputs and results once each (of the experts' weights those that some token is expected to reach), and
    the operations of the products, of a quantisation, of one exponential and the sums for each logit."""
    es = _BYTES[case["type"]]
    if case["family"] == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * (k * (es + 1) + 4 * _blocks(k)), "flops": 3 * m * k}
    if case["family"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + 4 * _blocks(k) * (m + _blocks(n)) + es * m * n, "flops": 2 * m * n * k}
    if case["family"] == "moe":
        t, e, top, h, i = case["t"], case["e"], case["top"], case["h"], case["i"]
        dense = 2 if case["type"] == "fp8" else es
        reached = e * (1 - (1 - top / e) ** t)
        scales = 4 * (_blocks(2 * i) * _blocks(h) + _blocks(h) * _blocks(i)) if case["type"] == "fp8" else 0
        return {"bytes": reached * (3 * h * i * es + scales) + dense * h * (e + 2 * t), "flops": 2 * t * h * (3 * top * i + e)}
    return {"bytes": case["b"] * (case["v"] * es + 24), "flops": 4 * case["b"] * case["v"]}


# ----------------------------------------------------------------- exact --
def _exact_e4m3(x):
    """The e4m3 value nearest to each 64-bit one (ties to even), |x| <= 448."""
    exponent = np.maximum(np.frexp(x)[1] - 1, -6)
    step = np.ldexp(1.0, exponent - 3)
    return np.rint(x / step) * step


def exact(case, seed):
    d = _inputs(case, seed)
    if case["family"] == "quantize":
        x = d["x"].double().cpu().numpy()
        starts = np.arange(0, case["k"], BLOCK)
        scale = np.maximum(np.maximum.reduceat(np.abs(x), starts, axis=1) / 448.0, 2.0 ** -126)
        return {"q": _exact_e4m3(x / np.repeat(scale, BLOCK, axis=1)[:, :case["k"]]), "scale": scale}
    if case["family"] == "gemm":
        y = 0
        for k0 in range(0, case["k"], BLOCK):
            rows = torch.arange(case["n"], device="cuda") // BLOCK
            part = d["a"][:, k0:k0 + BLOCK].double() @ d["b"][:, k0:k0 + BLOCK].double().t().contiguous()
            y = y + part * d["sa"][:, k0 // BLOCK].double()[:, None] * d["sb"][rows, k0 // BLOCK].double()[None, :]
        return {"y": y}
    if case["family"] == "moe":
        i, lines = case["i"], []

        def matrix(name, j):
            w = d[name][j].double()
            if case["type"] != "fp8":
                return w
            at = [torch.arange(n, device="cuda") // BLOCK for n in w.shape]
            return w * d[name + "_scale"][j].double()[at[0][:, None], at[1][None, :]]

        for x in d["x"].double():
            logits = (d["router"].double() @ x).cpu().numpy()
            chosen = np.lexsort((np.arange(case["e"]), -logits))[:case["top"]]
            share = np.exp(logits[chosen] - logits[chosen[0]])
            y = 0
            for j, s in zip(chosen, share / share.sum()):
                both = matrix("gate_up", int(j)) @ x
                y = y + s * (matrix("down", int(j)) @ (both[:i] / (1 + torch.exp(-both[:i])) * both[i:]))
            lines.append(y)
        return {"y": torch.stack(lines)}
    rows = {n: t.cpu().numpy().astype(np.float64) for n, t in d.items() if n != "logits"}
    tokens = []
    for r, logits in enumerate(d["logits"].double().cpu().numpy()):
        order = np.argsort(-logits, kind="stable")
        if not rows["temperature"][r] > 0:
            tokens.append(order[0])
            continue
        order = order[:int(rows["top_k"][r])] if rows["top_k"][r] >= 1 else order
        w = np.exp((logits[order] - logits[order[0]]) / rows["temperature"][r])
        n = len(order)
        if rows["top_p"][r] < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), rows["top_p"][r] * np.sum(w), side="left")))
        n = max(1, min(n, int(np.count_nonzero(w >= rows["min_p"][r]))))
        by_index = np.sort(order[:n])
        sums = np.cumsum(np.exp((logits[by_index] - logits[order[0]]) / rows["temperature"][r]))
        at = int(np.searchsorted(sums, rows["uniform"][r] * sums[-1], side="right"))
        tokens.append(by_index[min(at, n - 1)])
    return {"token": np.array(tokens, np.int32)}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(24)]:
        w = work(c)
        print("%-110s %10.3f MB %10.3f GFLOP" % (c, w["bytes"] / 1e6, w["flops"] / 1e9))
