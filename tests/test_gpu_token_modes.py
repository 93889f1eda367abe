"""Products whose exactness, NaN or infinities show which matrix instructions they pass through, and FLOAT32 operands of
experts and sampling in the precision modes."""
import numpy as np
import pytest

import token_ops_ref as R
from test_gpu_token_ops import check, expert_graph, expert_operands, expert_values, gemm_graph, sample_graph
from util import announce, run_hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 128), (7, 130, 200), (16, 96, 1040), (16, 4100, 384)])
def test_few_rows_lose_no_small_products(odla, kind, m, n, k):
    """Up to 16 rows are sums of exact products: eight terms of which two cancel, 200704 each, and six are 20."""
    announce("product %s %d x %d x %d beside cancelling products" % (kind, m, n, k))
    rng = np.random.default_rng(m + n + k)
    va, vb = np.zeros((m, k)), np.zeros((n, k))
    for at in range(0, k - 8, 128):
        at += 8 * int(rng.integers(0, (min(128, k - at) - 8) // 8 + 1))
        va[:, at:at + 8] = [448, 448, 5, 5, 5, 5, 5, 5]
        vb[:, at:at + 8] = [448, -448, 4, 4, 4, 4, 4, 4]
    a, b = R.e4m3_encode(va), R.e4m3_encode(vb)
    sa = rng.uniform(0.5, 2, (m, R.blocks(k))).astype(np.float32)
    sb = rng.uniform(0.5, 2, (R.blocks(n), R.blocks(k))).astype(np.float32)
    got = R.values(run_hip(gemm_graph(odla, kind, (a, sa), (b, sb)), {"a": a, "sa": sa, "b": b, "sb": sb})["y"], kind)
    x, w = R.row_values(a, sa), R.square_values(b, sb)
    want = x @ w.T
    off = (R.BLOCK + R.blocks(k) + 3) * R.UNIT * (np.abs(x) @ np.abs(w).T)
    check(got, want, off + R.EPS[kind] / 2 * (np.abs(want) + off) + R.LEAST[kind], "product", kind)
    assert np.all(off < np.abs(want) / 4)        # (what the 8-bit instructions would drop is all of it)


# rows of one wavefront's tiles, of a workgroup's, of tiles of 128 and of 256, and rows that are no whole vectors
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(9, 300, 272), (40, 300, 272), (150, 200, 260), (300, 300, 400), (1500, 1700, 272), (3500, 3500, 144), (4200, 1030, 136)])
def test_nan_and_infinite_scales_stay_in_their_row_or_column(odla, kind, m, n, k):
    announce("product %s %d x %d x %d with NaN codes, NaN and infinite scales" % (kind, m, n, k))
    rng = np.random.default_rng(m)
    a, b = rng.integers(0x28, 0x38, (m, k), dtype=np.uint8), rng.integers(0x28, 0x38, (n, k), dtype=np.uint8)    # (positive)
    sa = rng.uniform(0.01, 0.02, (m, R.blocks(k))).astype(np.float32)
    sb = rng.uniform(0.01, 0.02, (R.blocks(n), R.blocks(k))).astype(np.float32)
    a[2, k - 3], a[m - 1, 1] = 0x7f, 0xff
    b[5, 3], b[n - 1, k - 1] = 0xff, 0x7f
    sa[4, 1], sa[m - 2, 0] = np.nan, np.inf
    got = R.values(run_hip(gemm_graph(odla, kind, (a, sa), (b, sb)), {"a": a, "sa": sa, "b": b, "sb": sb})["y"], kind)
    nan = np.zeros((m, n), bool)
    nan[[2, m - 1, 4]] = True
    nan[:, [5, n - 1]] = True
    assert np.array_equal(np.isnan(got), nan)
    inf = np.zeros((m, n), bool)
    inf[m - 2] = ~nan[m - 2]
    assert np.array_equal(np.isinf(got), inf) and np.all(got[inf] > 0)


@pytest.mark.parametrize("mode", ["fp16", "bf16"])
@pytest.mark.parametrize("weights", ["fp32", "fp8"])
@pytest.mark.parametrize("t,e,h,i,top_k", [(1, 8, 64, 32, 2), (7, 12, 136, 100, 3), (40, 3, 72, 200, 2)])
def test_experts_of_float32_operands_in_a_mode(odla, mode, weights, t, e, h, i, top_k):
    """FLOAT32 operands are stored, and results rounded, as the mode says; the scales of 8-bit weights are not."""
    announce("experts of FLOAT32 operands in %s mode, %s weights" % (mode, weights))
    d = expert_operands(t, e, h, i, "fp32", weights, seed=t + e)
    if weights == "fp8":       # scales of which fp16 keeps a few bits, and activations that make up for them
        d["gate_up_scale"], d["x"] = d["gate_up_scale"] * np.float32(2.0 ** -10), d["x"] * np.float32(2.0 ** 10)
        d["router"] = d["router"] * np.float32(2.0 ** -10)
    got = run_hip(expert_graph(odla, d, top_k, "fp32", weights), d, repeats=2, **{mode: True})["y"]
    stored = {n: R.values(R.to_bits(v.astype(np.float64), mode), mode) if v.dtype == np.float32 and not n.endswith("scale") else v for n, v in d.items()}
    want, bound = R.experts(*expert_values(stored, "fp32", weights), top_k, True, 1.0, mode, weights == "fp8")
    check(got, want, bound, "experts", mode)


@pytest.mark.parametrize("mode", ["fp16", "bf16"])
def test_sampling_of_float32_logits_in_a_mode(odla, mode):
    """Logits are stored as the mode says, parameters are not."""
    announce("sampling of FLOAT32 logits in %s mode" % mode)
    rng = np.random.default_rng(9)
    n, v = 60, 3001
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    p = {"temperature": rng.choice([0.3, 1.0, 1.7], n), "top_k": rng.choice([0, 3, 700], n), "top_p": rng.choice([0.8, 0.9999, 1.0], n),
         "min_p": rng.choice([0.0, 0.0123], n), "uniform": rng.random(n)}
    feeds = {k: np.asarray(a, np.int32 if k == "top_k" else np.float32) for k, a in p.items()}
    got = run_hip(sample_graph(odla, "fp32", x.shape, {k: a.shape for k, a in feeds.items()}), {"logits": x, **feeds}, **{mode: True})["token"]
    stored = R.values(R.to_bits(x, mode), mode)
    want = [R.sample_row(stored[r], **{k: a[r] for k, a in feeds.items()}) for r in range(n)]
    assert np.array_equal(got, want)
