"""Operators of a decoder layer together, as a model runs them: norm with residual and 8-bit result, product, attention over the pages
of a cache, product, norm, experts, norm, logits, the chosen tokens and their log probabilities.  A prompt and then token after
token, two computations on one pair of caches; every operator's result against the formula on the operands that it was given."""
import threading

import numpy as np
import pytest

import layer_ops_ref as L
import token_ops_ref as R
import test_gpu_log_probs as log_probs
import test_gpu_rms_norm as norms
from test_gpu_token_ops import check, expert_operands
from util import announce

pytestmark = pytest.mark.gpu

E, HEADS, GROUP, D, PAGE, PAGES, VOCABULARY, WINDOW = 160, 2, 4, 96, 12, 24, 1000, 60
EPSILON = 1e-5
BETWEEN = ("n1", "n1s", "r1", "qkv", "y", "yq", "ys", "a", "n2", "r2", "moe", "n3", "n3s", "r3", "logits")


def weights(seed=5):
    rng = np.random.default_rng(seed)
    w = expert_operands(1, 6, E, 64, "bf16", "fp8", seed=seed)
    del w["x"]
    for n, rows, k in (("wqkv", (HEADS * GROUP + 2 * HEADS) * D, E), ("wo", E, HEADS * GROUP * D), ("head", VOCABULARY, E)):
        w[n], w[n + "_s"] = R.quantize_squares(rng.standard_normal((rows, k)) * k ** -0.5 * (4 if n == "head" else 1))
    for n in ("w1", "w2", "w3"):
        w[n] = R.to_bits(1 + 0.2 * rng.standard_normal(E), "bf16")
    w["embedding"] = R.to_bits(rng.standard_normal((VOCABULARY, E)), "bf16")
    return w


def layer(odla, w, t, between=True):
    """A builder of the step for t tokens of two sequences."""
    b = odla.HipBuilder()
    bf16, fp8 = odla.BFLOAT16, odla.FLOAT8_E4M3
    put = lambda n: b.const(n, w[n], {np.dtype(np.uint8): fp8, np.dtype(np.uint16): bf16}.get(w[n].dtype))
    norm = lambda x, r, n, names, dtype=None: b.rms_norm(x, put(n), r, EPSILON, dtype, names)
    v = {}
    x, r = b.arg("x", (t, E), bf16), b.arg("r", (t, E), bf16)
    v["n1"], v["n1s"], v["r1"] = norm(x, r, "w1", ("n1", "n1s", "r1"), fp8)
    v["qkv"] = b.block_gemm(v["n1"], v["n1s"], put("wqkv"), put("wqkv_s"), bf16, "qkv")
    part = lambda first, heads: b.reshape(b.slice(v["qkv"], (0, first * D), (t, (first + heads) * D)), (t, heads, D))
    cache = lambda n: b.arg(n, (PAGES, PAGE, HEADS, D), bf16)
    v["y"] = b.reshape(b.paged_attention(part(0, HEADS * GROUP), part(HEADS * GROUP, HEADS), part(HEADS * GROUP + HEADS, HEADS), cache("kc"), cache("vc"),
                                         b.arg("pt", (2, 10), np.int32), b.arg("n", (2,), np.int32), b.arg("s", (3,), np.int32), window=WINDOW, name="att"),
                       (t, HEADS * GROUP * D), "y")
    v["yq"], v["ys"] = b.block_quantize(v["y"], ("yq", "ys"))
    v["a"] = b.block_gemm(v["yq"], v["ys"], put("wo"), put("wo_s"), bf16, "a")
    v["n2"], v["r2"] = norm(v["a"], v["r1"], "w2", ("n2", "r2"))
    v["moe"] = b.mixture_of_experts(v["n2"], put("router"), put("gate_up"), put("down"), 2, put("gate_up_scale"), put("down_scale"), name="moe")
    v["n3"], v["n3s"], v["r3"] = norm(v["moe"], v["r2"], "w3", ("n3", "n3s", "r3"), fp8)
    v["logits"] = b.block_gemm(v["n3"], v["n3s"], put("head"), put("head_s"), np.float32, "logits")
    v["token"] = b.sample(v["logits"], b.arg("u", (t,)), b.const("temp", np.array([0.8], np.float32)), b.const("top_k", np.array([50], np.int32)), name="token")
    v["lp"], v["e"], v["tl"], v["tt"] = b.log_probs(v["logits"], v["token"], 4, ("lp", "e", "tl", "tt"))
    for n in (BETWEEN if between else ()) + ("token", "lp", "e", "tl", "tt"):
        b.output(v[n], n)
    return b


def check_layer(w, got, feeds, kc, vc):
    """kc, vc: the caches' bits before."""
    u = lambda a: R.values(a, "bf16")
    norms.check({"q": got["n1"], "scale": got["n1s"], "sum": got["r1"]}, {"x": feeds["x"], "r": feeds["r"], "w": w["w1"]}, "bf16", "bf16", EPSILON)
    check(u(got["qkv"]), *R.block_gemm(got["n1"], got["n1s"], w["wqkv"], w["wqkv_s"], "bf16"), "queries, keys and values")
    t = len(feeds["x"])
    q, k, v = (a.reshape(t, -1, D) for a in np.split(u(got["qkv"]), [HEADS * GROUP * D, (HEADS * GROUP + HEADS) * D], 1))
    y, bound, _, _ = L.paged_attention(q, k, v, u(kc), u(vc), feeds["pt"], feeds["n"], feeds["s"], D ** -0.5, WINDOW, "bf16")
    check(u(got["y"]), y.reshape(t, -1), bound.reshape(t, -1), "attention")
    yq, ys = R.quantize_rows(u(got["y"]))
    assert np.array_equal(got["yq"], yq) and np.array_equal(got["ys"], ys)
    check(u(got["a"]), *R.block_gemm(yq, ys, w["wo"], w["wo_s"], "bf16"), "product behind attention")
    norms.check({"y": got["n2"], "sum": got["r2"]}, {"x": got["a"], "r": got["r1"], "w": w["w2"]}, "bf16", "bf16", EPSILON)
    experts = [R.square_values(w[n], w[n + "_scale"]) for n in ("gate_up", "down")]
    check(u(got["moe"]), *R.experts(u(got["n2"]), u(w["router"]), *experts, 2, True, 1.0, "bf16", True), "experts")
    norms.check({"q": got["n3"], "scale": got["n3s"], "sum": got["r3"]}, {"x": got["moe"], "r": got["r2"], "w": w["w3"]}, "bf16", "bf16", EPSILON)
    check(got["logits"], *R.block_gemm(got["n3"], got["n3s"], w["head"], w["head_s"], "fp32"), "logits")
    want = [R.sample_row(l, np.float32(0.8), 50, 1.0, 0.0, x) for l, x in zip(got["logits"].astype(np.float64), feeds["u"])]
    assert np.array_equal(got["token"], np.array(want, np.int32))
    log_probs.check(got, got["logits"].astype(np.float64), got["token"].reshape(t, 1), 4)


class Sequences:
    """Two sequences, their pages and what is to be computed next."""

    def __init__(self, odla, w, new=(37, 5), cached=(0, 20), seed=1):
        rng = np.random.default_rng(seed)
        self.w, self.rng, self.new, self.cached = w, rng, list(new), list(cached)
        self.table = rng.permutation(PAGES)[:20].reshape(2, 10).astype(np.int32)
        start = lambda: R.to_bits(rng.standard_normal((PAGES, PAGE, HEADS, D)), "bf16")
        self.kc, self.vc = odla.DeviceArray(start()), odla.DeviceArray(start())
        self.tokens = rng.integers(0, VOCABULARY, sum(new))

    def feeds(self):
        t = sum(self.new)
        return {"x": self.w["embedding"][self.tokens], "r": R.to_bits(self.rng.standard_normal((t, E)), "bf16"), "kc": self.kc, "vc": self.vc, "pt": self.table,
                "n": np.array(self.cached, np.int32), "s": np.cumsum([0] + self.new).astype(np.int32), "u": self.rng.random(t).astype(np.float32)}

    def grow(self, got):
        ends = np.cumsum(self.new) - 1
        self.cached = [c + n for c, n in zip(self.cached, self.new)]
        self.tokens, self.new = got["token"][ends], [1, 1]

    def close(self):
        self.kc.close()
        self.vc.close()


@pytest.mark.parametrize("graph", [True, False])
def test_a_prompt_and_its_tokens(odla, graph, monkeypatch):
    announce("a prompt and its tokens, %s" % ("captured" if graph else "launch by launch"))
    monkeypatch.setenv("ODLA_HIP_GRAPH_MIN_STEPS", "1")
    w = weights()
    q = Sequences(odla, w)
    builders, sessions = [], []
    # the prompt, a token, and a token of which nothing between is kept: other places in memory
    for t, between in ((sum(q.new), True), (2, True), (2, False)):
        builders.append(layer(odla, w, t, between))
        sessions.append(builders[-1].session(use_graph=graph))      # (a context is of the computation that was made last)
    try:
        for step in range(5):
            feeds, before = q.feeds(), (q.kc.get(), q.vc.get())
            s = sessions[min(step, 1)]
            got = s.run(feeds)
            check_layer(w, got, feeds, *before)
            after = q.kc.get(), q.vc.get()
            assert not np.array_equal(after[0], before[0])
            for _ in range(3):       # the same tokens to the same places: the same bits
                again = s.run(feeds)
                assert all(np.array_equal(again[n], got[n]) for n in got)
                if step:
                    only = sessions[2].run(feeds)
                    assert all(np.array_equal(only[n], got[n]) for n in only)
            assert np.array_equal(q.kc.get(), after[0]) and np.array_equal(q.vc.get(), after[1])
            q.grow(got)
    finally:
        [s.close() for s in sessions]
        [b.destroy() for b in builders]
        q.close()


def test_two_contexts_on_two_threads(odla):
    """Two contexts of one computation, each with its caches, at once."""
    announce("two contexts of a layer's step side by side")
    w = weights()
    b = layer(odla, w, 2)
    both = [Sequences(odla, w, (1, 1), cached, seed=3 + i) for i, cached in enumerate([(70, 1), (0, 110)])]
    feeds, before = [q.feeds() for q in both], [(q.kc.get(), q.vc.get()) for q in both]
    sessions = [b.session(), b.session()]
    got = [[], []]
    try:
        def work(i):
            for _ in range(20):
                got[i].append(sessions[i].run(feeds[i]))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        for i in range(2):
            assert len(got[i]) == 20
            check_layer(w, got[i][0], feeds[i], *before[i])
            for g in got[i]:
                assert all(np.array_equal(g[n], got[i][0][n]) for n in g)
    finally:
        [s.close() for s in sessions]
        b.destroy()
        [q.close() for q in both]
