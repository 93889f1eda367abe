"""odla_hip_LogProbs against the formulas in 64 bits: sizes, types, ties, odd values, precision modes."""
import numpy as np
import pytest

import layer_ops_ref as L
import token_ops_ref as R
from test_gpu_token_ops import np_kind
from util import announce, run_hip, run_hip_stored

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]


def graph(odla, kind, shape, per_row, top):
    lead = shape[:-1]

    def build(b):
        tokens = b.arg("t", lead + ((per_row,) if per_row > 1 or not lead else ()), np.int32)
        names = ("lp", "e", "tl", "tt")
        for v, n in zip(b.log_probs(b.arg("l", shape, np_kind(odla, kind)), tokens, top, names), names):
            b.output(v, n)
    return build


def run_and_check(odla, kind, bits, tokens, top, **kw):
    """bits [.., V], tokens [rows, n]"""
    shape = bits.shape
    rows, per_row = tokens.shape
    lead = shape[:-1]
    got = run_hip(graph(odla, kind, shape, per_row, top), {"l": bits, "t": tokens.reshape(lead + ((per_row,) if per_row > 1 or not lead else ())).astype(np.int32)}, **kw)
    check(got, R.values(bits, kind).reshape(rows, -1), tokens, top)
    return got


def check(got, logits, tokens, top):
    rows = len(logits)
    lp, lpb, ent, entb, tl, tb, ti = L.log_probs(logits, tokens, top)

    def near(have, want, bound, what):
        have = np.asarray(have, np.float64).reshape(want.shape)
        same = have == want
        with np.errstate(invalid="ignore"):
            off = np.abs(have - want)
        assert np.all(same | (off <= bound)), "%s: worst %g of %g" % (what, np.nanmax(np.where(same, 0, off)), np.max(bound))

    near(got["lp"], lp, lpb, "log p")
    near(got["e"], ent, entb, "entropy")
    if top:
        assert np.array_equal(got["tt"].reshape(rows, top), ti)
        near(got["tl"], tl, tb, "alternatives")


def logits_of(shape, kind, seed, spread=3.0):
    rng = np.random.default_rng(seed)
    return R.to_bits(rng.standard_normal(shape) * spread, kind)


# one part of 8192 (narrow) and of 32768 logits (wide), both ends, and rows of several parts
SIZES = [1, 2, 7, 8, 63, 257, 1000, 8192, 8193, 20001, 32768, 32769, 65544, 100003]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v", SIZES)
def test_rows_of_all_lengths(odla, kind, v):
    announce("log probabilities of %d logits, %s" % (v, kind))
    rng = np.random.default_rng(v)
    rows = 3
    for top in sorted({0, 1, min(v, 5), min(v, 32)}):
        run_and_check(odla, kind, logits_of((rows, v), kind, v), rng.integers(0, v, (rows, 2)), top)


@pytest.mark.parametrize("shape,per_row", [((5000, 33), 1), ((2, 3, 500), 4), ((999,), 1), ((999,), 64), ((70, 9000), 64), ((300, 33000), 1)])
def test_shapes(odla, shape, per_row):
    announce("log probabilities %s, %d tokens a row" % (shape, per_row))
    rows = int(np.prod(shape[:-1])) if len(shape) > 1 else 1
    tokens = np.random.default_rng(1).integers(0, shape[-1], (rows, per_row))
    run_and_check(odla, "bf16", logits_of(shape, "bf16", 3), tokens, 3, repeats=3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v", [1, 9, 2048, 2056, 4095, 5001])
def test_many_rows(odla, kind, v):
    """1100 rows are streamed by a wavefront each: some with equal, infinite and missing logits and nearly certain tokens."""
    announce("log probabilities of 1100 rows of %d logits, %s" % (v, kind))
    rng = np.random.default_rng(v)
    x = rng.standard_normal((1100, v)) * 3
    x[0] = -np.inf
    x[1] = 0.5
    x[2, ::3] = np.nan
    x[3] = np.inf
    x[4, v // 2] = np.inf
    x[5, v // 2] = 60.0
    x[6, -1] = 30.0
    x[7] = -np.inf
    x[7, v // 3] = -5.0
    x[8] = {"fp32": -3e38, "fp16": -65504.0, "bf16": -3e38}[kind]
    x[9] = np.sort(x[9])                  # the maximum grows all along
    x[10] = np.sort(x[10])[::-1]
    x[11, ::2] = -np.inf
    x[12] = np.nan
    tokens = rng.integers(0, v, (1100, 2))
    tokens[:20, 0] = v // 2
    run_and_check(odla, kind, R.to_bits(x, kind), tokens, 0)


def test_the_longest_row(odla):
    announce("log probabilities of 524288 logits")
    run_and_check(odla, "fp32", logits_of((2, 524288), "fp32", 3), np.array([[0, 524287], [5, 9]]), 32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v", [500, 9000, 70000])
def test_equal_logits(odla, kind, v):
    """Ties go to the lowest index, also where thousands of logits reach the bound."""
    announce("log probabilities of equal logits, %s, %d" % (kind, v))
    rng = np.random.default_rng(2)
    x = np.zeros((6, v))
    x[1] = -7.5
    x[2] = rng.integers(0, 3, v)
    x[3, rng.integers(0, v, 40)] = 9
    x[4] = np.where(np.arange(v) % 2, 0.0, -0.0)
    x[5] = -np.arange(v) % 16
    run_and_check(odla, kind, R.to_bits(x, kind), rng.integers(0, v, (6, 3)), 20)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v", [40, 9000, 70000])
def test_odd_values(odla, kind, v):
    announce("log probabilities of infinite and missing logits, %s, %d" % (kind, v))
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, v))
    x[0] = -np.inf
    x[1, 3::2] = -np.inf
    x[2, 7] = np.nan
    x[3, [4, 30]] = np.inf
    x[4] = -np.inf
    x[4, 11] = 2.5                       # a certain token
    x[5] = np.nan
    x[6] = {"fp32": -3e38, "fp16": -65504.0, "bf16": -3e38}[kind]
    x[6, 9] = 0.0
    x[7] = np.finfo(np.float32).min if kind == "fp32" else x[6, 0]     # all of the type's lowest value
    x[8, 0] = 40.0                       # nearly certain: what is left over counts
    tokens = np.stack([np.full(9, 11), np.full(9, 30), np.full(9, 7), np.full(9, -1), np.full(9, v), np.full(9, 9), np.zeros(9, int), np.full(9, 2 ** 31 - 1)], 1)
    run_and_check(odla, kind, R.to_bits(x, kind), tokens, 8)


def test_nearly_certain_tokens_keep_their_digits(odla):
    """log p of a token beside which 1e-9 is left: to parts in a million of itself, not of 1."""
    announce("log probabilities of nearly certain tokens")
    for v in (1000, 40000):
        x = np.full((1, v), -30.0)
        x[0, 5] = 0.0
        got = run_and_check(odla, "fp32", x.astype(np.float32), np.array([[5]]), 2)
        want = -np.log1p((v - 1) * np.exp(-30.0))
        assert abs(got["lp"][0] - want) <= 1e-5 * abs(want)


@pytest.mark.parametrize("mode", [{"fp16": True}, {"bf16": True}])
def test_precision_modes(odla, mode):
    """FLOAT32 logits are stored as the mode says; what comes out is fp32, also behind operators that move elements."""
    announce("log probabilities of FLOAT32 logits, %s" % mode)
    kind = "fp16" if "fp16" in mode else "bf16"
    bits = logits_of((4, 600), kind, 9)
    x = R.values(bits, kind).astype(np.float32)
    tokens = np.random.default_rng(3).integers(0, 600, (4, 1))

    def build(b):
        got = b.log_probs(b.arg("l", x.shape), b.arg("t", (4,), np.int32), 3)
        for v, n in zip(got, ("lp", "e", "tl", "tt")):
            b.output(v, n)
        b.output(b.reshape(got[0], (2, 2)), "lp2")
    got = run_hip(build, {"l": x, "t": tokens[:, 0].astype(np.int32)}, **mode)
    check(got, R.values(bits, kind), tokens, 3)
    assert np.array_equal(got["lp2"].reshape(-1), got["lp"])


def test_stored(odla, tmp_path):
    announce("log probabilities, stored and loaded")
    feeds = {"l": logits_of((3, 40000), "bf16", 1), "t": np.array([1, 2, 3], np.int32)}
    build = graph(odla, "bf16", (3, 40000), 1, 7)
    a, b = run_hip(build, feeds), run_hip_stored(build, feeds, str(tmp_path / "score.odla"))
    for n in a:
        assert np.array_equal(a[n], b[n]), n


def test_log_p_of_a_drawn_token(odla):
    """What odla_hip_Sample draws goes straight into odla_hip_LogProbs; a row with nothing to draw gives -inf."""
    announce("a token is drawn and scored")
    bits = logits_of((6, 3000), "fp32", 7)
    bits[4] = -np.inf

    def build(b):
        l = b.arg("l", bits.shape)
        t = b.sample(l, b.arg("u", (6,)), top_k=b.const("k", np.array([50], np.int32)), name="t")
        b.output(t, "t")
        for v, n in zip(b.log_probs(l, t, 4), ("lp", "e", "tl", "tt")):
            b.output(v, n)
    got = run_hip(build, {"l": bits, "u": np.random.default_rng(1).random(6).astype(np.float32)}, repeats=2)
    assert got["t"][4] == -1 and got["lp"][4] == -np.inf
    check(got, bits.astype(np.float64), got["t"][:, None], 4)
