"""A computation with operators of a token step gives the same bits in every execution: it is not run as two half
batches, whose products have other last bits, and with them other tokens."""
import numpy as np
import pytest

import token_ops_ref as R
from test_gpu_token_ops import expert_graph, expert_operands
from util import announce, run_hip

pytestmark = pytest.mark.gpu


def both(monkeypatch, build, feeds):
    monkeypatch.setenv("ODLA_HIP_BATCH_SPLIT", "0")
    whole = run_hip(build, feeds)
    monkeypatch.setenv("ODLA_HIP_BATCH_SPLIT", "2")
    again = run_hip(build, feeds, repeats=2)
    for n in whole:
        assert np.array_equal(whole[n], again[n]), n


def test_a_product_of_32_rows_stays_whole(odla, monkeypatch):
    """32 rows pass through the 8-bit matrix instructions, 16 as bf16."""
    announce("a product and a token of 32 rows, halves asked for")
    rng = np.random.default_rng(6)
    x = R.to_bits(rng.standard_normal((32, 1000)) * 10.0 ** rng.integers(-2, 3, (32, 1000)), "bf16")
    w, ws = R.quantize_squares(rng.standard_normal((500, 1000)))

    def build(b):
        q, s = b.block_quantize(b.arg("x", x.shape, odla.BFLOAT16))
        y = b.block_gemm(q, s, b.const("w", w, odla.FLOAT8_E4M3), b.const("ws", ws), odla.BFLOAT16, name="y")
        b.output(y, "y")
        b.output(b.sample(y, b.arg("u", (32,)), name="t"), "t")
    both(monkeypatch, build, {"x": x, "u": rng.random(32).astype(np.float32)})


def test_experts_of_32_tokens_stay_whole(odla, monkeypatch):
    """32 tokens for three experts are taken 64 at a time, 16 eight at a time: other orders of the sums."""
    announce("experts of 32 tokens, halves asked for")
    d = expert_operands(32, 3, 3000, 400, "bf16", "bf16", seed=12)
    both(monkeypatch, lambda b: expert_graph(odla, d, 1, "bf16", "bf16", const=True)(b), {"x": d["x"]})
