"""Operators of a token step against 64-bit references: block quantisation, block-scaled product, mixture of
experts, sampling; alone over sizes, types and odd values, and as one run behind each other."""
import numpy as np
import pytest

import token_ops_ref as R
from util import announce, run_hip, run_hip_stored

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]


def np_kind(odla, kind):
    return {"fp32": np.float32, "fp16": np.float16, "bf16": odla.BFLOAT16, "fp8": odla.FLOAT8_E4M3}[kind]


def check(got, want, bound, what, kind="fp32"):
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    # (a value that rounds beyond the type becomes its infinity: fp16's from 65520 on)
    ok = (off <= bound) | (np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + bound >= 65520) & (kind == "fp16"))
    assert np.all(ok), "%s: %d of %d values off, worst %g of its bound" % (what, np.sum(~ok), ok.size, np.max(off / bound))


# -------------------------------------------------------------- quantisation --
def quantize_graph(odla, kind, shape):
    def build(b):
        q, s = b.block_quantize(b.arg("x", shape, np_kind(odla, kind)), names=("q", "s"))
        b.output(q, "q")
        b.output(s, "s")
    return build


def same_codes(a, b):
    """Equal bit patterns; the two of NaN are one."""
    nan = (a & 127) == 127
    return np.array_equal(nan, (b & 127) == 127) and np.array_equal(a[~nan], b[~nan])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 129), (5, 127), (2, 3, 256), (17, 640), (300, 8), (64, 1023), (130,), (1025, 136)])
def test_quantized_rows(odla, kind, shape):
    announce("block quantisation %s %s" % (kind, shape))
    rng = np.random.default_rng(sum(shape))
    x = rng.standard_normal(shape) * 10.0 ** rng.integers(-3, 4, shape[:-1] + (1,))
    x[..., ::37] *= 50
    bits = R.to_bits(x, kind)
    got = run_hip(quantize_graph(odla, kind, shape), {"x": bits})
    q, s = R.quantize_rows(R.values(bits, kind))
    assert np.array_equal(got["s"], s)
    assert same_codes(got["q"], q)
    # against the formula in 64 bits: half a step of 2^-3, or half the subnormal step of 2^-9, and the scale's own rounding
    # (fp16 values that became infinite in the conversion of the inputs are the next test's)
    v = R.values(bits, kind)
    with np.errstate(invalid="ignore"):
        off = np.abs(R.row_values(got["q"], got["s"]) - v)
    each = np.repeat(got["s"].astype(np.float64), R.BLOCK, axis=-1)[..., :shape[-1]]
    assert np.all(np.isinf(each) | (off <= (2.0 ** -4 + 2.0 ** -23) * np.abs(v) + 2.0 ** -10 * (1 + 2.0 ** -20) * each))


@pytest.mark.parametrize("kind", KINDS)
def test_quantized_rows_of_odd_values(odla, kind):
    announce("block quantisation of zeros, subnormals, infinities and NaN, %s" % kind)
    x = np.zeros((7, 200))
    x[1, 3] = R.LEAST[kind] * 3
    x[2] = np.linspace(-1, 1, 200)
    x[2, 7] = np.nan
    x[3, 130] = np.inf
    x[4, 130] = -np.inf
    x[5] = -0.0
    x[6] = {"fp32": 3.0e38, "fp16": 65504.0, "bf16": 3.0e38}[kind]
    bits = R.to_bits(x, kind)
    got = run_hip(quantize_graph(odla, kind, x.shape), {"x": bits})
    with np.errstate(invalid="ignore"):
        q, s = R.quantize_rows(R.values(bits, kind))
    assert np.array_equal(got["s"], s)
    have = R.e4m3_decode(got["q"])
    assert same_codes(got["q"], q)
    assert np.isnan(have[2, 7]) and np.isnan(have[2]).sum() == 1     # a NaN stays alone
    assert np.isinf(got["s"][3, 1]) and np.isfinite(got["s"][3, 0])


def test_every_8_bit_value_is_its_own_quantisation(odla):
    announce("block quantisation of the values of the type")
    v = R.e4m3_decode(np.arange(256))
    v = np.where(np.isnan(v), 448.0, v)
    rows = np.stack([np.concatenate([np.full(1, 448.0), v[:127]]), np.concatenate([np.full(1, 448.0), v[128:255]])])
    got = run_hip(quantize_graph(odla, "fp32", rows.shape), {"x": rows.astype(np.float32)})
    assert np.all(got["s"] == 1.0)
    assert np.array_equal(R.e4m3_decode(got["q"]), rows)


# ------------------------------------------------------------------- product --
def gemm_graph(odla, kind, a, b, const=False):
    def build(g):
        m = a[0].shape
        x, xs = g.arg("a", m, odla.FLOAT8_E4M3), g.arg("sa", a[1].shape)
        w = g.const("b", b[0], odla.FLOAT8_E4M3) if const else g.arg("b", b[0].shape, odla.FLOAT8_E4M3)
        ws = g.const("sb", b[1]) if const else g.arg("sb", b[1].shape)
        g.output(g.block_gemm(x, xs, w, ws, np_kind(odla, kind), name="y"), "y")
    return build


def gemm_operands(m, n, k, seed, lead=()):
    rng = np.random.default_rng(seed)
    a = R.quantize_rows(rng.standard_normal(lead + (m, k)) * 10.0 ** rng.integers(-2, 3, lead + (m, 1)))
    b = R.quantize_squares(rng.standard_normal((n, k)))
    b = (b[0], (b[1] * 10.0 ** rng.uniform(-2, 2, b[1].shape)).astype(np.float32))
    return a, b


GEMM_SIZES = [(1, 1, 1), (1, 16, 128), (1, 130, 129), (2, 3, 15), (5, 128, 256), (16, 257, 384), (17, 96, 1040), (31, 250, 100),
              (33, 64, 2049), (48, 384, 512), (64, 129, 640), (65, 128, 128), (100, 100, 100), (127, 255, 272), (129, 1, 300),
              (200, 515, 130), (256, 256, 256), (300, 130, 1000), (513, 140, 384), (7, 2000, 96), (1, 300, 5000),
              (260, 768, 1296), (515, 1030, 400), (1030, 514, 272)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_block_product(odla, kind, m, n, k):
    announce("block product %s %d x %d x %d" % (kind, m, n, k))
    a, b = gemm_operands(m, n, k, seed=m * 7 + n * 3 + k)
    got = run_hip(gemm_graph(odla, kind, a, b), {"a": a[0], "sa": a[1], "b": b[0], "sb": b[1]})["y"]
    want, bound = R.block_gemm(*a, *b, kind)
    check(R.values(got, kind), want, bound, "product", kind)


@pytest.mark.parametrize("m,n,k", [(3, 140, 260), (70, 130, 392)])
def test_block_product_with_constant_weights_and_leading_extents(odla, m, n, k):
    announce("block product, constants, rank 3: %d x %d x %d" % (m, n, k))
    a, b = gemm_operands(m, n, k, seed=5, lead=(2,))
    got = run_hip(gemm_graph(odla, "fp32", a, b, const=True), {"a": a[0], "sa": a[1]}, repeats=3)["y"]
    want, bound = R.block_gemm(*a, *b, "fp32")
    assert got.shape == (2, m, n)
    check(got, want, bound, "product")


@pytest.mark.parametrize("m", [4, 150])
def test_a_nan_stays_in_its_row_or_column(odla, m):
    announce("block product with NaN, %d rows" % m)
    a, b = gemm_operands(m, 150, 260, seed=11)
    a[0][2, 200] = 0x7f
    b[0][5, 3] = 0xff
    got = run_hip(gemm_graph(odla, "fp32", a, b), {"a": a[0], "sa": a[1], "b": b[0], "sb": b[1]})["y"]
    nan = np.zeros(got.shape, bool)
    nan[2] = True
    nan[:, 5] = True
    assert np.array_equal(np.isnan(got), nan)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_quantized_rows_of_every_magnitude(odla, kind):
    """Blocks whose scales pass the borders between the two ways of dividing, each with values down to subnormals."""
    announce("block quantisation of blocks of every magnitude, %s" % kind)
    rng = np.random.default_rng(21)
    exponents = np.array([-130, -118, -75, -71, -70, -69, -62, -61, -60, -20, 0, 60, 110, 118, 119, 127])
    x = (1 + rng.random((len(exponents), 384))) * rng.choice([-1.0, 1.0], (len(exponents), 384)) / 2
    x *= 2.0 ** rng.choice([0, -1, -5, -9, -12, -40], x.shape)
    x = np.ldexp(x, exponents[:, None])
    x[:, 5], x[:, 6], x[:, 130] = -0.0, 0.0, -2.0 ** -149
    bits = R.to_bits(x, kind)
    got = run_hip(quantize_graph(odla, kind, x.shape), {"x": bits})
    q, s = R.quantize_rows(R.values(bits, kind))
    assert np.array_equal(got["s"], s) and same_codes(got["q"], q)



@pytest.mark.parametrize("mode", ["fp32", "fp16", "bf16"])
def test_quantised_in_front_of_a_product(odla, mode):
    """FLOAT32 values as the precision mode stores them; the scales stay fp32 between the two operators."""
    announce("quantisation and product in %s mode" % mode)
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((9, 300)) * 1e-3).astype(np.float32)
    w, ws = R.quantize_squares(rng.standard_normal((200, 300)))
    ws = (ws * 1e-3).astype(np.float32)           # (below what fp16 scales could hold)

    def build(b):
        q, s = b.block_quantize(b.arg("x", x.shape), names=("q", "s"))
        b.output(s, "s")
        b.output(b.block_gemm(q, s, b.const("w", w, odla.FLOAT8_E4M3), b.const("ws", ws), name="y"), "y")

    got = run_hip(build, {"x": x}, fp16=mode == "fp16", bf16=mode == "bf16", repeats=2)
    q, s = R.quantize_rows(R.values(R.to_bits(x, mode), mode))
    assert np.array_equal(got["s"], s)
    want, bound = R.block_gemm(q, s, w, ws, mode)
    check(got["y"], want, bound, "product")


def test_8_bit_values_are_moved_as_they_are(odla):
    announce("moving 8-bit values")
    rng = np.random.default_rng(1)
    x = rng.integers(0, 256, (6, 40), dtype=np.uint8)
    idx = np.array([4, 0, 4], np.int32)

    def build(b):
        v = b.arg("x", x.shape, odla.FLOAT8_E4M3)
        b.output(b.reshape(v, (3, 80), name="r"), "r")
        b.output(b.transpose(v, (1, 0), name="t"), "t")
        b.output(b.slice(v, (1, 3), (5, 37), (2, 1), name="s"), "s")
        b.output(b.concat([v, v], 1, name="c"), "c")
        b.output(b.gather(v, b.const("i", idx), 0, name="g"), "g")

    got = run_hip(build, {"x": x})
    assert np.array_equal(got["r"], x.reshape(3, 80)) and np.array_equal(got["t"], x.T)
    assert np.array_equal(got["s"], x[1:5:2, 3:37]) and np.array_equal(got["c"], np.concatenate([x, x], 1))
    assert np.array_equal(got["g"], x[idx])


# ------------------------------------------------------------------- experts --
def expert_operands(t, e, h, i, kind, weights, seed):
    rng = np.random.default_rng(seed)
    d = {"x": R.to_bits(rng.standard_normal((t, h)), kind), "router": R.to_bits(rng.standard_normal((e, h)) * 2 * h ** -0.5, kind)}
    gu, dn = rng.standard_normal((e, 2 * i, h)) * h ** -0.5, rng.standard_normal((e, h, i)) * i ** -0.5
    if weights == "fp8":
        d["gate_up"], d["gate_up_scale"] = R.quantize_squares(gu)
        d["down"], d["down_scale"] = R.quantize_squares(dn)
    else:
        d["gate_up"], d["down"] = R.to_bits(gu, kind), R.to_bits(dn, kind)
    return d


def expert_values(d, kind, weights):
    if weights == "fp8":
        return (R.values(d["x"], kind), R.values(d["router"], kind), R.square_values(d["gate_up"], d["gate_up_scale"]),
                R.square_values(d["down"], d["down_scale"]))
    return tuple(R.values(d[n], kind) for n in ("x", "router", "gate_up", "down"))


def expert_graph(odla, d, top_k, kind, weights, renormalize=True, scaling=1.0, const=False):
    types = {n: np_kind(odla, weights if n in ("gate_up", "down") else kind) for n in ("x", "router", "gate_up", "down")}
    types["gate_up_scale"] = types["down_scale"] = np.float32

    def build(b):
        put = lambda n: (b.const(n, d[n], types[n] if isinstance(types[n], odla.ElementType) else None) if const and n != "x"
                         else b.arg(n, d[n].shape, types[n]))
        v = {n: put(n) for n in d}
        b.output(b.mixture_of_experts(v["x"], v["router"], v["gate_up"], v["down"], top_k, v.get("gate_up_scale"),
                                      v.get("down_scale"), renormalize, scaling, name="y"), "y")
    return build


EXPERT_SIZES = [(1, 1, 1, 1, 1), (1, 8, 64, 32, 2), (2, 5, 33, 17, 3), (3, 16, 128, 48, 1), (7, 40, 130, 100, 6), (16, 6, 256, 64, 6),
                (17, 4, 96, 130, 2), (33, 9, 200, 72, 4), (40, 3, 64, 200, 3), (1, 300, 64, 16, 32), (5, 64, 136, 24, 8), (70, 2, 40, 33, 1),
                (1, 33, 520, 264, 4)]


@pytest.mark.parametrize("kind,weights", [("fp32", "fp32"), ("fp16", "fp16"), ("bf16", "bf16"), ("bf16", "fp8"), ("fp16", "fp8"), ("fp32", "fp8")])
@pytest.mark.parametrize("t,e,h,i,top_k", EXPERT_SIZES)
def test_experts(odla, kind, weights, t, e, h, i, top_k):
    announce("experts %s / %s: %d tokens, %d of %d experts, %d x %d" % (kind, weights, t, top_k, e, h, i))
    d = expert_operands(t, e, h, i, kind, weights, seed=t + 10 * e + h + i)
    renormalize, scaling = (t + e) % 2 == 0, 1.0 if t % 3 else 2.5
    got = run_hip(expert_graph(odla, d, top_k, kind, weights, renormalize, scaling), d)["y"]
    want, bound = R.experts(*expert_values(d, kind, weights), top_k, renormalize, scaling, kind, weights == "fp8")
    check(R.values(got, kind), want, bound, "experts")


@pytest.mark.parametrize("kind,weights", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp8"), ("fp32", "fp8")])
@pytest.mark.parametrize("t,e,h,i,top_k", [(64, 64, 72, 200, 4), (64, 40, 72, 330, 2), (200, 16, 272, 152, 3), (300, 4, 136, 104, 2), (65, 1, 64, 600, 1),
                                           (2, 2, 33100, 20, 2), (3, 1, 24, 33040, 1), (40, 2, 33040, 10, 2), (8, 1024, 40, 8, 32)])
def test_experts_of_many_tiles_columns_and_steps(odla, kind, weights, t, e, h, i, top_k):
    """More tiles than resident workgroups, more columns than a tile has, rows of more than 64 steps a wavefront."""
    announce("experts %s / %s: %d tokens, %d of %d experts, %d x %d" % (kind, weights, t, top_k, e, h, i))
    d = expert_operands(t, e, h, i, kind, weights, seed=t + 10 * e + h + i)
    got = R.values(run_hip(expert_graph(odla, d, top_k, kind, weights), d, repeats=2)["y"], kind)
    x, router, gate_up, down = expert_values(d, kind, weights)
    sure = np.ones(t, bool)
    if top_k < e:       # (tokens whose choice is clear)
        order = np.sort(x @ router.T, 1)
        sure = order[:, -top_k] - order[:, -top_k - 1] > 4.1 * (h + 2) * R.UNIT * (np.abs(x) @ np.abs(router).T).max(1)
        assert sure.sum() >= 0.75 * t
    want, bound = R.experts(x[sure], router, gate_up, down, top_k, True, 1.0, kind, weights == "fp8")
    check(got[sure], want, bound, "experts")


def test_experts_with_constant_weights_and_leading_extents(odla):
    announce("experts, constants, rank 3")
    d = expert_operands(10, 12, 144, 80, "bf16", "fp8", seed=77)
    want, bound = R.experts(*expert_values(d, "bf16", "fp8"), 3, True, 1.0, "bf16", True)
    d["x"] = d["x"].reshape(2, 5, 144)
    got = run_hip(expert_graph(odla, d, 3, "bf16", "fp8", const=True), {"x": d["x"]}, repeats=3)["y"]
    assert got.shape == (2, 5, 144)
    check(R.values(got, "bf16").reshape(10, 144), want, bound, "experts")


def test_equal_router_rows_take_the_lowest_experts(odla):
    announce("experts with equal logits")
    d = expert_operands(4, 70, 64, 32, "fp32", "fp32", seed=9)
    d["router"][:] = d["router"][0]
    d["router"][3] = -d["router"][0]
    got = run_hip(expert_graph(odla, d, 5, "fp32", "fp32"), d)["y"]
    x, router, gate_up, down = expert_values(d, "fp32", "fp32")
    for r in range(4):
        front = x[r] @ router[3] > x[r] @ router[0]
        logits = np.full(70, 1.0)
        logits[3] = 2.0 if front else 0.0
        chosen = np.lexsort((np.arange(70), -logits))[:5]
        l = x[r] @ router[chosen].T
        w = np.exp(l - l.max())
        want = sum(s * (down[j] @ ((g := gate_up[j, :32] @ x[r]) / (1 + np.exp(-g)) * (gate_up[j, 32:] @ x[r]))) for j, s in zip(chosen, w / w.sum()))
        assert np.max(np.abs(got[r] - want)) <= 1e-4 * np.max(np.abs(want))


def test_a_token_with_nan_does_not_touch_the_others(odla):
    announce("experts with a NaN token")
    d = expert_operands(20, 6, 72, 40, "fp32", "fp32", seed=21)
    clean = run_hip(expert_graph(odla, d, 2, "fp32", "fp32"), d)["y"]
    d["x"] = d["x"].copy()
    d["x"][4, 5] = np.nan
    d["x"][9, :] = np.inf
    got = run_hip(expert_graph(odla, d, 2, "fp32", "fp32"), d)["y"]
    assert np.all(np.isnan(got[4])) and np.all(np.isnan(got[9]))
    keep = [r for r in range(20) if r not in (4, 9)]
    assert np.array_equal(got[keep], clean[keep])


def test_experts_of_many_tokens(odla):
    announce("experts of 512 tokens, 1024 experts")
    d = expert_operands(512, 1024, 32, 16, "bf16", "bf16", seed=4)
    d["router"][:, :] = R.to_bits(np.random.default_rng(8).standard_normal((1024, 32)) * 4, "bf16")
    got = R.values(run_hip(expert_graph(odla, d, 2, "bf16", "bf16"), d)["y"], "bf16")
    x, router, gate_up, down = expert_values(d, "bf16", "bf16")
    logits = x @ router.T
    order = np.sort(logits, 1)
    sure = order[:, -2] - order[:, -3] > 4 * 34 * R.UNIT * (np.abs(x) @ np.abs(router).T).max(1)   # (the choice is clear)
    assert sure.sum() > 400
    want, bound = R.experts(x[sure], router, gate_up, down, 2, True, 1.0, "bf16")
    check(got[sure], want, bound, "experts")


# -------------------------------------------------------------------- sampling --
PARAMS = ("temperature", "top_k", "top_p", "min_p", "uniform")


def sample_graph(odla, kind, shape, have):
    def build(b):
        rows = {n: b.arg(n, s, np.int32 if n == "top_k" else np.float32) for n, s in have.items()}
        b.output(b.sample(b.arg("logits", shape, np_kind(odla, kind)), name="token", **rows), "token")
    return build


def run_sample(odla, kind, logits, p, **kw):
    feeds = {n: np.asarray(v, np.int32 if n == "top_k" else np.float32) for n, v in p.items()}
    got = run_hip(sample_graph(odla, kind, logits.shape, {n: v.shape for n, v in feeds.items()}), {"logits": logits, **feeds}, **kw)["token"]
    v = R.values(logits, kind).reshape(-1, logits.shape[-1])
    want = [R.sample_row(v[r], **{n: a.reshape(-1)[r if a.size > 1 else 0] for n, a in feeds.items()}) for r in range(len(v))]
    return got, np.array(want, np.int32).reshape(got.shape)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (5, 63), (7, 64), (6, 65), (9, 1000), (4, 1025), (12, 4096), (5, 12345), (3, 50257), (2, 131072)])
def test_sampled_tokens(odla, kind, rows, v):
    announce("sampling %s %d x %d" % (kind, rows, v))
    rng = np.random.default_rng(rows * 1000 + v)
    x = rng.standard_normal((rows, v)) * 3
    x[rng.random((rows, v)) < 0.02] = -np.inf
    x[:, v // 2] = 0.5
    p = {"temperature": rng.choice([0.0, 0.3, 1.0, 1.7], rows), "top_k": rng.choice([0, 1, 3, 40, 1000, v], rows),
         "top_p": rng.choice([0.1, 0.8, 0.95, 1.0], rows), "min_p": rng.choice([0.0, 0.02, 0.3], rows), "uniform": rng.random(rows)}
    got, want = run_sample(odla, kind, R.to_bits(x, kind), p)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p", None])
def test_each_parameter_alone_and_single_ones(odla, only):
    announce("sampling with %s alone" % only)
    rng = np.random.default_rng(17)
    x = (rng.standard_normal((40, 777)) * 2).astype(np.float32)
    p = {"uniform": rng.random(40)}
    if only is not None:
        p[only] = {"temperature": rng.random(40) + 0.2, "top_k": rng.integers(0, 60, 40), "top_p": rng.random(40), "min_p": rng.random(40) * 0.3}[only]
    got, want = run_sample(odla, "fp32", x, p)
    assert np.array_equal(got, want)
    single = {n: np.asarray(a).reshape(-1)[:1] for n, a in p.items()}     # one element serves every row
    got, want = run_sample(odla, "fp32", x.reshape(4, 10, 777), single)
    assert got.shape == (4, 10) and np.array_equal(got, want)


def test_rows_that_leave_little(odla):
    """Rows without anything to draw, with one token, with infinities, NaN and equal logits; parameters beyond their ranges."""
    announce("sampling from odd rows")
    nan, inf, v = np.nan, np.inf, 300
    rows, p = [], {n: [] for n in PARAMS}

    def row(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.5):
        rows.append(np.broadcast_to(np.asarray(x, np.float32), (v,)))
        for n, a in zip(PARAMS, (temperature, top_k, top_p, min_p, uniform)):
            p[n].append(a)

    ramp = np.linspace(-4, 4, v)
    alone = np.full(v, -inf)
    alone[211] = -3e38
    row(-inf); row(nan); row(alone); row(alone, top_k=5, top_p=0.5, uniform=0.999); row(alone, temperature=0.0)
    some = np.full(v, -3.4028235e38, np.float32)      # (a mask of the type's lowest value)
    some[[3, 70, 299]] = [1.0, 2.0, 1.5]
    for u in (0.0, 0.2, 0.45, 0.7, 0.99999994, 1.0):
        row(some, uniform=u)
        row(some, uniform=u, temperature=inf)
    top = ramp.copy(); top[[9, 200]] = inf
    row(top, uniform=0.2); row(top, uniform=0.8); row(top, temperature=0.0); row(top, temperature=inf, uniform=0.8)
    holes = ramp.copy(); holes[::3] = nan
    row(holes, uniform=0.9); row(holes, top_k=2, uniform=0.9); row(holes, temperature=nan)
    for u in (0.0, 0.31, 0.77, 0.999):                # all equal: ties go by index
        row(1.25, uniform=u); row(1.25, top_k=7, uniform=u); row(1.25, top_p=0.1, uniform=u); row(1.25, top_k=100, top_p=0.25, uniform=u)
        row(np.where(np.arange(v) % 2, 0.0, -0.0), top_k=9, uniform=u)
    for k in (-5, 0, 1, v - 1, v, v + 1, 2 ** 31 - 1):
        row(ramp, top_k=k, uniform=0.001)
    for t in (-1.0, 0.0, 1e-40, 1e-30, 1e-3, 1e30):
        row(ramp, temperature=t, uniform=0.3)
    for t in (-0.5, 0.0, 1e-30, 0.5, 1.0, 1.5, nan):
        row(ramp, top_p=t, uniform=0.6)
        row(ramp, min_p=t, uniform=0.6)
        row(ramp[::-1], top_p=t, min_p=0.1, top_k=20, uniform=0.6)
    row(ramp, uniform=nan); row(ramp, uniform=-1.0); row(ramp, uniform=2.0)
    got, want = run_sample(odla, "fp32", np.stack(rows), p)
    assert np.array_equal(got, want), [(i, int(g), int(w)) for i, (g, w) in enumerate(zip(got, want)) if g != w]
    assert got[0] == -1 and got[1] == -1 and got[2] == 211


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("v", [300, 6001, 70000])
def test_rows_with_infinite_logits(odla, kind, v):
    """Only the infinite ones are drawn, alike, whatever the cuts leave of them."""
    announce("sampling %s from %d logits with infinite ones" % (kind, v))
    rng = np.random.default_rng(v)
    p = {n: [] for n in PARAMS}
    for k in (0, 1, 2, 3, 4, 20, 2500):
        for top_p in (1.0, 0.6, 0.3):
            for min_p, temperature in ((0.0, 1.0), (0.5, 0.3), (0.0, np.inf)):
                for n, a in zip(PARAMS, (temperature, k, top_p, min_p, rng.random())):
                    p[n].append(a)
    rows = len(p["top_k"])
    x = rng.standard_normal((rows, v)) * 4
    x[:, ::7] = -np.inf
    x[:, 5] = {"fp32": 3.4028234e38, "fp16": 65504.0, "bf16": 3.3895e38}[kind]
    for r in range(rows):
        x[r, rng.choice(v, 3, replace=False)] = np.inf
    got, want = run_sample(odla, kind, R.to_bits(x, kind), p)
    assert np.array_equal(got, want), [(i, int(g), int(w)) for i, (g, w) in enumerate(zip(got, want)) if g != w]


def test_drawn_frequencies_follow_the_weights(odla):
    """Evenly spaced random numbers hit every token by its share of the sum, to one draw."""
    announce("sampling frequencies")
    x = np.log(np.array([1.0, 2.0, 3.0, 4.0, 6.0])).astype(np.float32)
    n = 1600
    p = {"uniform": (np.arange(n) + 0.5) / n}
    got, want = run_sample(odla, "fp32", np.broadcast_to(x, (n, 5)).copy(), p)
    assert np.array_equal(got, want)
    assert np.all(np.abs(np.bincount(got, minlength=5) - n * np.array([1, 2, 3, 4, 6]) / 16) <= 1)


@pytest.mark.parametrize("v", [6, 2051])
def test_rows_of_equal_logits_in_16_bits(odla, v):
    announce("sampling from few distinct logits, %d" % v)
    rng = np.random.default_rng(v)
    x = R.to_bits(rng.integers(-2, 3, (60, v)).astype(float), "bf16")
    p = {"top_k": rng.integers(0, v, 60), "top_p": rng.random(60), "uniform": rng.random(60)}
    got, want = run_sample(odla, "bf16", x, p)
    assert np.array_equal(got, want)


# ------------------------------------------------------------- as they are used --
def token_step(odla, d, head, rows, batch=-1):
    """Experts, a classifier with 8-bit weights and the choice of a token."""
    def build(b):
        n = batch if batch > 0 else len(rows["uniform"])
        x = b.arg("x", (batch if batch < 0 else n, d["x"].shape[1]), odla.BFLOAT16)
        y = b.mixture_of_experts(x, b.const("router", d["router"], odla.BFLOAT16), b.const("gate_up", d["gate_up"], odla.FLOAT8_E4M3),
                                 b.const("down", d["down"], odla.FLOAT8_E4M3), 3, b.const("gs", d["gate_up_scale"]),
                                 b.const("ds", d["down_scale"]), name="moe")
        q, s = b.block_quantize(y, names=("q", "qs"))
        logits = b.block_gemm(q, s, b.const("head", head[0], odla.FLOAT8_E4M3), b.const("hs", head[1]), np.float32, name="logits")
        b.output(y, "moe")
        b.output(logits, "logits")
        b.output(b.sample(logits, b.arg("uniform", (batch if batch < 0 else n,)), b.const("t", np.array([0.7], np.float32)),
                          b.const("k", np.array([40], np.int32)), b.const("p", np.array([0.9], np.float32)), name="token"), "token")
    return build


def step_inputs(n, seed=31):
    d = expert_operands(n, 10, 160, 96, "bf16", "fp8", seed=seed)
    head = R.quantize_squares(np.random.default_rng(2).standard_normal((1500, 160)))
    return d, head, {"uniform": np.random.default_rng(3).random(n).astype(np.float32)}


def check_step(got, d, head, rows):
    y, bound = R.experts(*expert_values(d, "bf16", "fp8"), 3, True, 1.0, "bf16", True)
    check(R.values(got["moe"], "bf16"), y, bound, "experts")
    q, s = R.quantize_rows(R.values(got["moe"], "bf16"))
    logits, bound = R.block_gemm(q, s, *head, "fp32")
    check(got["logits"], logits, bound, "logits")
    # (the temperature is an fp32 value)
    want = [R.sample_row(l, np.float32(0.7), 40, np.float32(0.9), 0.0, u) for l, u in zip(got["logits"].astype(np.float64), rows["uniform"])]
    assert np.array_equal(got["token"], np.array(want, np.int32))


@pytest.mark.parametrize("graph", [True, False])
def test_a_token_step(odla, graph, monkeypatch):
    announce("a token step, %s" % ("captured" if graph else "launch by launch"))
    monkeypatch.setenv("ODLA_HIP_GRAPH_MIN_STEPS", "1")
    d, head, rows = step_inputs(6)
    got = run_hip(token_step(odla, d, head, rows, 6), {"x": d["x"], **rows}, use_graph=graph, repeats=4)
    check_step(got, d, head, rows)


def test_a_stored_token_step(odla, tmp_path):
    announce("a stored token step")
    d, head, rows = step_inputs(4)
    build = token_step(odla, d, head, rows, 4)
    want = run_hip(build, {"x": d["x"], **rows})
    got = run_hip_stored(build, {"x": d["x"], **rows}, str(tmp_path / "step.odla"))
    for n in want:
        assert np.array_equal(got[n], want[n]), n


def test_a_token_step_at_every_batch(odla):
    announce("a token step at several batches")
    d, head, rows = step_inputs(8)
    hb = odla.HipBuilder(max_batch=8)
    try:
        token_step(odla, d, head, rows, -1)(hb)
        s = hb.session()
        try:
            for n in (8, 3, 1, 8):
                s.set_batch(n)
                part = {"uniform": rows["uniform"][:n]}
                check_step(s.run({"x": d["x"][:n], **part}), {**d, "x": d["x"][:n]}, head, part)
        finally:
            s.close()
    finally:
        hb.destroy()


def test_a_token_step_without_allocation(odla):
    announce("a token step in the static scratch")
    d, head, rows = step_inputs(5)
    hb = odla.HipBuilder()
    try:
        token_step(odla, d, head, rows, 5)(hb)
        s = hb.session()
        try:
            s.bind_device_io({"x": d["x"], **rows})
            s.execute()
            want = s.fetch_device_outputs()
            for _ in range(2):
                assert s.execute_static() == 0
                got = s.fetch_device_outputs()
                for n in want:
                    assert np.array_equal(got[n], want[n]), n
        finally:
            s.close()
    finally:
        hb.destroy()
    check_step(want, d, head, rows)


def test_two_contexts_of_one_step_on_two_threads(odla):
    announce("two contexts of a token step side by side")
    import threading
    d, head, rows = step_inputs(6)
    hb = odla.HipBuilder()
    try:
        token_step(odla, d, head, rows, 6)(hb)
        sessions = [hb.session(), hb.session()]
        feeds = [{"x": d["x"], **rows}, {"x": d["x"][::-1].copy(), "uniform": rows["uniform"][::-1].copy()}]
        try:
            alone = [s.run(f) for s, f in zip(sessions, feeds)]
            got = [[], []]

            def work(k):
                for _ in range(20):
                    got[k].append(sessions[k].run(feeds[k]))

            threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
            [t.start() for t in threads]
            [t.join() for t in threads]
            for k in range(2):
                assert len(got[k]) == 20
                for g in got[k]:
                    for n in g:
                        assert np.array_equal(g[n], alone[k][n]), n
        finally:
            [s.close() for s in sessions]
    finally:
        hb.destroy()
    check_step(alone[0], d, head, rows)


def test_results_reach_only_their_rows(odla):
    """Device buffers larger than the results: what stands behind them stays."""
    announce("buffers behind the results")
    import ctypes
    L = odla.load_library()
    d, head, rows = step_inputs(3)
    hb = odla.HipBuilder()
    try:
        token_step(odla, d, head, rows, 3)(hb)
        s = hb.session()
        held = []
        try:
            s.bind_device_io({"x": d["x"], **rows})
            guard = np.full(4096, 0xa5, np.uint8)
            for name, (h, shape, dt) in hb.outs.items():
                n = int(np.prod(shape)) * dt.itemsize
                p = ctypes.c_void_p()
                assert L.odla_AllocateDeviceMemory(ctypes.byref(p), n + guard.nbytes) == 0
                assert L.odla_CopyMemory(ctypes.c_void_p(p.value + n), guard.ctypes.data_as(ctypes.c_void_p), guard.nbytes, odla.ODLA_MEMCPY_H2D) == 0
                assert L.odla_BindToOutput(h, p, s.ctx) == 0
                held.append((p, n, name, shape, dt))
            s.execute()
            got = {}
            for p, n, name, shape, dt in held:
                raw = np.empty(n + guard.nbytes, np.uint8)
                assert L.odla_CopyMemory(raw.ctypes.data_as(ctypes.c_void_p), p, raw.nbytes, odla.ODLA_MEMCPY_D2H) == 0
                assert np.array_equal(raw[n:], guard), name
                got[name] = raw[:n].view(dt).reshape(shape)
        finally:
            for p, *_ in held:
                L.odla_FreeDeviceMemory(p)
            s.close()
    finally:
        hb.destroy()
    check_step(got, d, head, rows)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("spread", [0.0, 1e-6, 0.02, 1.0, 30.0])
def test_cuts_in_crowded_and_empty_places(odla, kind, spread):
    """Rows from all equal to far apart, cuts from the first element to the last: few, thousands or all beside the cut."""
    announce("sampling with spread %g, %s" % (spread, kind))
    rng = np.random.default_rng(5)
    v, n = 9001, 36
    x = 3.0 + spread * rng.standard_normal((n, v))
    x[1::3, rng.integers(0, v, 40)] += 4.0
    p = {"temperature": np.tile([0.5, 1.0, 20.0], n // 3), "top_k": np.tile(np.repeat([0, 2, 45, 1500, 4500, 9000], 3), n // 18),
         "top_p": np.tile([1.0, 0.3, 0.97, 0.9999], n // 4), "min_p": np.tile([0.0, 0.0, 0.001], n // 3), "uniform": rng.random(n)}
    got, want = run_sample(odla, kind, R.to_bits(x, kind), p)
    assert np.array_equal(got, want), [(i, int(g), int(w)) for i, (g, w) in enumerate(zip(got, want)) if g != w]


def test_the_largest_vocabulary(odla):
    announce("sampling from 524288 logits")
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((6, 1 << 19)) * 2).astype(np.float32)
    p = {"top_k": [0, 0, 50, 5000, 0, 200000], "top_p": [1.0, 0.9, 0.9, 1.0, 0.999, 0.5], "min_p": [0, 0, 0, 0, 0.01, 0], "uniform": rng.random(6)}
    got, want = run_sample(odla, "fp32", x, p)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(3500, 3500, 400), (4100, 3080, 128), (257, 49000, 272), (1500, 1700, 400), (1161, 2305, 128), (130, 12000, 1040)])
def test_block_product_of_many_tiles(odla, kind, m, n, k):
    """Sizes that give (most of) the compute units a tile of 256 x 256, or of 128 x 128; checked on rows and columns across the edges of tiles."""
    announce("block product %s %d x %d x %d" % (kind, m, n, k))
    rng = np.random.default_rng(m + n)
    a = (rng.integers(0, 256, (m, k), dtype=np.uint8) & 0xbf, rng.uniform(0.5, 2, (m, R.blocks(k))).astype(np.float32))
    b = (rng.integers(0, 256, (n, k), dtype=np.uint8) & 0xbf, rng.uniform(0.001, 0.1, (R.blocks(n), R.blocks(k))).astype(np.float32))
    got = R.values(run_hip(gemm_graph(odla, kind, a, b), {"a": a[0], "sa": a[1], "b": b[0], "sb": b[1]})["y"], kind)
    rows = np.unique(np.concatenate([np.arange(0, m, 97), [m - 1, 255, 256], np.arange(120, 136)]))
    rows = rows[rows < m]
    for at in (slice(0, 300), slice(n - 300, n)):
        cols = np.arange(n)[at]
        bb = b[0][cols]
        want = R.row_values(a[0][rows], a[1][rows]) @ (R.e4m3_decode(bb) * np.repeat(b[1][cols // R.BLOCK], R.BLOCK, axis=1)[:, :k]).T
        big = np.abs(R.row_values(a[0][rows], a[1][rows])) @ np.abs(R.e4m3_decode(bb) * np.repeat(b[1][cols // R.BLOCK], R.BLOCK, axis=1)[:, :k]).T
        # eight products: all but the largest lose up to 2^-13 of it; sums in fp32; the result's own rounding
        bound = (7 * 2.0 ** -13 + (R.BLOCK + R.blocks(k) + 3) * R.UNIT) * big + R.EPS[kind] / 2 * np.abs(want) * (1 + 2.0 ** -9)
        check(got[rows][:, cols], want, bound, "product", kind)
