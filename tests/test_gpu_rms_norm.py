"""odla_hip_RmsNorm against the formula in 64 bits: lengths, types, residuals, 8-bit results, odd values, precision modes."""
import numpy as np
import pytest

import layer_ops_ref as L
import token_ops_ref as R
from test_gpu_token_ops import np_kind, same_codes
from util import announce, run_hip, run_hip_stored

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]
EPSILON = 1e-5


def graph(odla, kind, shape, weight=None, residual=False, quantize=False, epsilon=EPSILON):
    def build(b):
        names = (["q", "scale"] if quantize else ["y"]) + (["sum"] if residual else [])
        got = b.rms_norm(b.arg("x", shape, np_kind(odla, kind)), None if weight is None else b.arg("w", shape[-1:], np_kind(odla, weight)),
                         b.arg("r", shape, np_kind(odla, kind)) if residual else None, epsilon, odla.FLOAT8_E4M3 if quantize else np_kind(odla, kind), names)
        for v, n in zip(got, names):
            b.output(v, n)
    return build


def feeds_of(shape, kind, weight, residual, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape) * 10.0 ** rng.integers(-2, 3, shape[:-1] + (1,))
    x[..., ::37] *= 30
    feeds = {"x": R.to_bits(x, kind)}
    if weight is not None:
        feeds["w"] = R.to_bits(1 + 0.3 * rng.standard_normal(shape[-1]), weight)
    if residual:
        feeds["r"] = R.to_bits(rng.standard_normal(shape), kind)
    return feeds


def check(got, feeds, kind, weight, epsilon=EPSILON):
    """Every result against the formula on the operands that were given."""
    v = {n: R.values(a, weight if n == "w" else kind) for n, a in feeds.items()}
    want, total = L.rms_norm(v["x"], v.get("r"), v.get("w"), epsilon)
    slack = L.norm_slack(want.shape[-1])
    if "sum" in got:
        assert np.all(np.abs(R.values(got["sum"], kind) - total) <= (R.EPS[kind] / 2 + 2 * L.ULP) * np.abs(total) + R.LEAST[kind])
    if "y" in got:
        off = np.abs(R.values(got["y"], kind) - want)
        assert np.all(off <= (R.EPS[kind] / 2 + slack) * np.abs(want) + R.LEAST[kind]), np.max(off)
        return
    k = want.shape[-1]
    for at in range(0, k, R.BLOCK):
        most = np.abs(want[..., at:at + R.BLOCK]).max(-1)
        scale = got["scale"][..., at // R.BLOCK].astype(np.float64)
        assert np.all(np.abs(scale - np.maximum(most / 448, 2.0 ** -126)) <= (slack + 2 * L.ULP) * scale)
    off = np.abs(R.row_values(got["q"], got["scale"]) - want)
    each = np.repeat(got["scale"].astype(np.float64), R.BLOCK, axis=-1)[..., :k]
    assert np.all(off <= (2.0 ** -4 + 2 * slack) * np.abs(want) + 2.0 ** -10 * (1 + 2.0 ** -20) * each)


# every form of the kernel by length (whole groups of eight and not), both ends of each, and the edges of a block
LENGTHS = [1, 7, 8, 127, 128, 129, 505, 512, 513, 1024, 1031, 2048, 2050, 4096, 4097, 8192, 8200, 32768, 32769, 40000, 65543]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", LENGTHS)
def test_rows_of_all_lengths(odla, kind, k):
    announce("norm of %d values, %s" % (k, kind))
    shape = (3, k)
    for residual, quantize in ((False, False), (True, True)):
        feeds = feeds_of(shape, kind, kind, residual, k)
        check(run_hip(graph(odla, kind, shape, kind, residual, quantize), feeds), feeds, kind, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("weight", [None, "fp32", "own"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("quantize", [False, True])
def test_operands_and_results(odla, kind, weight, residual, quantize):
    announce("norm %s weight %s residual %s 8-bit %s" % (kind, weight, residual, quantize))
    weight = kind if weight == "own" else weight
    for shape in ((1, 384), (2, 3, 130), (261, 72), (40,), (1000, 1)):
        feeds = feeds_of(shape, kind, weight, residual, sum(shape))
        check(run_hip(graph(odla, kind, shape, weight, residual, quantize), feeds, repeats=3), feeds, kind, weight)


@pytest.mark.parametrize("kind", KINDS)
def test_quantised_as_the_quantisation_does(odla, kind):
    """fp32 results quantised by odla_hip_BlockQuantize are what the norm quantises: the same codes and scales."""
    announce("norm with its own and with a separate quantisation")
    shape = (5, 700)
    feeds = feeds_of(shape, "fp32", "fp32", True, 4)

    def build(b):
        x, w, r = b.arg("x", shape), b.arg("w", (700,)), b.arg("r", shape)
        for v, n in zip(b.rms_norm(x, w, r, EPSILON, odla.FLOAT8_E4M3), ("q", "s", "z")):
            b.output(v, n)
        for v, n in zip(b.block_quantize(b.rms_norm(x, w, r, EPSILON)[0]), ("q2", "s2")):
            b.output(v, n)
    got = run_hip(build, feeds)
    assert np.array_equal(got["s"], got["s2"]) and same_codes(got["q"], got["q2"])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", [64, 200, 3001])
def test_rows_of_odd_values(odla, kind, k):
    announce("norm of zeros, subnormals, infinities and NaN, %s, %d" % (kind, k))
    x = np.ones((6, k))
    x[0] = 0
    x[1] = R.LEAST[kind] * 3
    x[2, 5] = np.nan
    x[3, 5] = np.inf
    x[4] = {"fp32": 1e15, "fp16": 60000.0, "bf16": 1e15}[kind]
    x[5, 1:] = 0
    feeds = {"x": R.to_bits(x, kind)}
    v = R.values(feeds["x"], kind)
    got = run_hip(graph(odla, kind, x.shape, quantize=True), feeds)
    want, _ = L.rms_norm(v, None, None, EPSILON)
    have = R.row_values(got["q"], got["scale"])
    assert np.all(have[0] == 0) and np.all(got["scale"][0] == np.float32(2.0 ** -126))
    assert np.all(np.isnan(have[2])) and np.isnan(have[3, 5]) and np.isnan(have[3]).sum() == 1
    y = R.values(run_hip(graph(odla, kind, x.shape), feeds)["y"], kind)
    for row in (0, 1, 4, 5):
        assert np.all(np.abs(y[row] - want[row]) <= (R.EPS[kind] / 2 + L.norm_slack(k)) * np.abs(want[row]) + R.LEAST[kind]), row
    assert np.all(np.isnan(y[2])) and np.isnan(y[3, 5]) and np.all(y[3, 6:] == 0)
    zero = R.values(run_hip(graph(odla, kind, x.shape, epsilon=0.0), feeds)["y"], kind)
    assert np.all(np.isnan(zero[0])) and np.all(np.isfinite(zero[4]))


@pytest.mark.parametrize("mode,kind", [({"fp16": True}, "fp16"), ({"bf16": True}, "bf16"), ({"bf16": "accuracy"}, "fp32")])
def test_precision_modes(odla, mode, kind):
    """FLOAT32 operands are stored as the mode says; the scales stay fp32."""
    announce("norm of FLOAT32 operands, %s" % mode)
    shape = (9, 520)
    feeds = feeds_of(shape, kind, kind, True, 3)
    feeds = {n: R.values(a, kind).astype(np.float32) for n, a in feeds.items()}      # (values that the mode's type holds)
    got = run_hip(graph(odla, "fp32", shape, "fp32", True, True), feeds, **mode)
    as_kind = {n: R.to_bits(a, kind) for n, a in feeds.items()}
    check({"q": got["q"], "scale": got["scale"], "sum": R.to_bits(got["sum"], kind)}, as_kind, kind, kind)
    assert np.array_equal(R.values(R.to_bits(got["sum"], kind), kind).astype(np.float32), got["sum"])


def test_a_sum_that_nothing_reads(odla):
    announce("norm with a residual, its sum unread, and one whose sum goes on")
    shape = (4, 96)
    feeds = feeds_of(shape, "bf16", "bf16", True, 8)

    def build(b):
        x, w, r = (b.arg(n, s, odla.BFLOAT16) for n, s in (("x", shape), ("w", (96,)), ("r", shape)))
        b.output(b.rms_norm(x, w, r, EPSILON)[0], "y")
        b.output(b.rms_norm(b.rms_norm(x, w, r, EPSILON)[1], w, None, EPSILON)[0], "y2")
    got = run_hip(build, feeds, repeats=3)
    check({"y": got["y"]}, feeds, "bf16", "bf16")
    v = {n: R.values(a, "bf16") for n, a in feeds.items()}
    want, _ = L.rms_norm(R.values(R.to_bits(v["x"] + v["r"], "bf16"), "bf16"), None, v["w"], EPSILON)
    assert np.all(np.abs(R.values(got["y2"], "bf16") - want) <= (R.EPS["bf16"] / 2 + L.norm_slack(96)) * np.abs(want) + R.LEAST["bf16"])


def test_stored(odla, tmp_path):
    announce("norm, stored and loaded")
    shape = (4, 300)
    feeds = feeds_of(shape, "fp16", "fp16", True, 8)
    build = graph(odla, "fp16", shape, "fp16", True, True)
    a, b = run_hip(build, feeds), run_hip_stored(build, feeds, str(tmp_path / "norm.odla"))
    for n in a:
        assert np.array_equal(a[n], b[n]), n


def test_rows_do_not_depend_on_their_number(odla):
    announce("norm of 1 and of 50 rows")
    feeds = feeds_of((50, 2000), "bf16", "bf16", True, 2)
    many = run_hip(graph(odla, "bf16", (50, 2000), "bf16", True, True), feeds)
    one = run_hip(graph(odla, "bf16", (1, 2000), "bf16", True, True), {"x": feeds["x"][7:8], "r": feeds["r"][7:8], "w": feeds["w"]})
    for n in many:
        assert np.array_equal(many[n][7:8], one[n]), n


@pytest.mark.parametrize("mode,kind", [({"fp16": True}, "bf16"), ({"bf16": True}, "fp16")])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("constant", [False, True])
def test_float32_weight_of_an_input_in_the_other_16_bit_type(odla, mode, kind, quantize, constant):
    """The mode stores FLOAT32 values in one 16-bit type, the input has the other: the weight stays fp32."""
    announce("norm of %s rows with a FLOAT32 weight, %s, 8-bit %s, constant %s" % (kind, mode, quantize, constant))
    for shape in ((3, 384), (2, 1001)):
        feeds = feeds_of(shape, kind, "fp32", True, shape[1])

        def build(b):
            names = (["q", "scale"] if quantize else ["y"]) + ["sum"]
            x, r = (b.arg(n, shape, np_kind(odla, kind)) for n in "xr")
            w = b.const("w", feeds["w"]) if constant else b.arg("w", shape[-1:])
            for v, n in zip(b.rms_norm(x, w, r, EPSILON, odla.FLOAT8_E4M3 if quantize else np_kind(odla, kind), names), names):
                b.output(v, n)
        check(run_hip(build, feeds, **mode), feeds, kind, "fp32")
