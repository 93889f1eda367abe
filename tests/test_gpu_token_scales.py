"""Scales and sampling parameters keep their fp32 bits behind moving operators in every precision mode."""
import numpy as np
import pytest

import token_ops_ref as R
import token_scale_graphs as G
from test_gpu_token_ops import check
from util import announce, run_hip

pytestmark = pytest.mark.gpu

MODES = {"fp32": {}, "fp16": {"fp16": True}, "bf16": {"bf16": True}}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("move", list(G.MOVES))
def test_moved_scales_reach_a_product(odla, move, mode):
    """Scales that 16 bits lose: near 1e-9 in front of the product (fp16 has nothing there), of full length (bf16)."""
    announce("scales behind %s, %s mode" % (move, mode))
    x, w, ws = G.moved_operands()
    x = (x.astype(np.float32) * np.float32(2.0 ** -10)).astype(np.float16)      # scales near 1e-6
    ws = (ws * np.float32(3e4)).astype(np.float32)
    got = run_hip(G.moved_product(odla, move, w, ws, outputs=True), {"x": x}, repeats=2, **MODES[mode])
    q, s = R.quantize_rows(x)
    q, s = G.ROWS[move](q), G.ROWS[move](s)
    assert np.array_equal(got["ms"], s)
    want, bound = R.block_gemm(q, s, w, ws, "fp16")
    check(got["y"], want, bound, "product", "fp16")
    # a product of two scales is stored as the mode says: each factor and the result rounded once
    eps = R.EPS[mode]
    s = s.astype(np.float64)
    off = np.abs(got["twice"].astype(np.float64) - s * s)
    assert np.all(off <= 2 * eps * s * s + 2 * s * R.LEAST[mode] + 2 * R.LEAST[mode])


@pytest.mark.parametrize("mode", ["fp16", "bf16"])
def test_scales_far_below_fp16(odla, mode):
    announce("scales near 1e-9, %s mode" % mode)
    x, w, ws = G.moved_operands()
    q, s = R.quantize_rows(x)
    s = (s * np.float32(1e-7)).astype(np.float32)
    ws = (ws * np.float32(1e8)).astype(np.float32)

    def build(b):
        sa = b.reshape(b.slice(b.arg("s", (6, 3)), (0, 0), (6, 3)), (6, 3))
        b.output(b.block_gemm(b.arg("q", q.shape, odla.FLOAT8_E4M3), sa, b.const("w", w, odla.FLOAT8_E4M3), b.const("ws", ws), np.float16, name="y"), "y")
    got = run_hip(build, {"q": q, "s": s}, **MODES[mode])["y"]
    want, bound = R.block_gemm(q, s, w, ws, "fp16")
    assert np.abs(want).max() > 1
    check(got, want, bound, "product", "fp16")


@pytest.mark.parametrize("mode", list(MODES))
def test_moved_parameters_reach_the_sampling(odla, mode):
    """Random numbers that differ in their last bits only: 16 bits of them would give one token."""
    announce("sampling parameters behind Slice and Reshape, %s mode" % mode)
    n, v = 64, 64
    p = np.zeros((3, n), np.float32)
    p[0] = np.float32(0.5) + (np.arange(n) - n // 2) * np.float32(2.0 ** -20)
    p[1], p[2] = 1.0, 0.99999
    logits = np.zeros((n, v), np.float16)
    logits[:, 0] = logits[:, 1] = 15.0

    def build(b):
        a = b.arg("p", (3, n))
        part = lambda i: b.reshape(b.slice(a, (i, 0), (i + 1, n)), (n,))
        b.output(b.sample(b.arg("l", (n, v), np.float16), part(0), temperature=part(1), top_p=part(2), name="t"), "t")
    got = run_hip(build, {"p": p, "l": logits}, **MODES[mode])["t"]
    want = [R.sample_row(logits[0], 1.0, 0, p[2, i], 0.0, p[0, i]) for i in range(n)]
    assert np.array_equal(got, want) and len(set(want)) > 1


MOVED_PARAMETERS = {
    "tile": lambda b, a, n: b.tile(b.slice(a, (n // 2,), (n // 2 + 1,)), (n,)),
    "broadcast": lambda b, a, n: b.broadcast_to(b.slice(a, (1,), (2,)), (n,)),
    "pad": lambda b, a, n: b.pad(b.slice(a, (0,), (n - 3,)), (1,), (2,)),
    "gather_elements": lambda b, a, n: b.gather_elements(a, b.const(None, np.arange(n, dtype=np.int32)[::-1].copy()), 0),
    "compress": lambda b, a, n: b.slice(b.compress(b.concat([a, a], 0), b.const(None, np.arange(2 * n) % 2 == 1), 0, (2 * n,)), (0,), (n,)),
}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("move", list(MOVED_PARAMETERS))
def test_random_numbers_keep_their_bits_on_the_way(odla, move, mode):
    announce("random numbers behind %s, %s mode" % (move, mode))
    n = 64
    u = np.float32(0.5) + (np.arange(n) - n // 2 - 0.5).astype(np.float32) * np.float32(2.0 ** -20)
    at = {"tile": np.full(n, n // 2), "broadcast": np.full(n, 1), "pad": np.clip(np.arange(n) - 1, 0, None), "gather_elements": np.arange(n)[::-1],
          "compress": np.concatenate([np.arange(1, n, 2)] * 2)}[move]
    moved = u[at].copy()
    if move == "pad":
        moved[[0, n - 2, n - 1]] = 0.0
    logits = np.full((n, 64), -np.inf, np.float32)
    logits[:, [3, 40]] = 1.0

    def build(b):
        b.output(b.sample(b.arg("l", logits.shape, np.float16), MOVED_PARAMETERS[move](b, b.arg("u", (n,)), n), name="t"), "t")
    got = run_hip(build, {"u": u, "l": logits.astype(np.float16)}, **MODES[mode])["t"]
    want = np.where(moved < 0.5, 3, 40)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("mode", list(MODES))
def test_scales_joined_with_computed_ones(odla, mode):
    """A Concat of moved scales, which stay fp32, and of ones that a group of element-wise operators made as the mode stores them."""
    announce("moved and computed scales in one Concat, %s mode" % mode)
    x, w, ws = G.moved_operands()

    def build(b):
        q, s = b.block_quantize(b.arg("x", x.shape, np.float16))
        made = b.mul(b.mul(b.slice(s, (0, 1), (6, 3)), b.const(None, np.array([[2.0]], np.float32))), b.const(None, np.array([[0.25]], np.float32)))
        sa = b.concat([b.slice(s, (0, 0), (6, 1)), made], 1)
        b.output(b.block_gemm(q, sa, b.const("w", w, odla.FLOAT8_E4M3), b.const("ws", ws), np.float16, name="y"), "y")
        b.output(sa, "sa")
    got = run_hip(build, {"x": x}, **MODES[mode])
    q, s = R.quantize_rows(x)
    want = s.copy()
    want[:, 1:] = R.values(R.to_bits(s[:, 1:].astype(np.float64), mode), mode) / 2      # (factors of two: one rounding)
    assert np.array_equal(got["sa"], want)
    y, bound = R.block_gemm(q, want, w, ws, "fp16")
    check(got["y"], y, bound, "product", "fp16")
