"""Sampling where differences of logits or their quotients with the temperature leave fp32."""
import numpy as np
import pytest

import token_ops_ref as R
from test_gpu_token_ops import run_sample
from util import announce

pytestmark = pytest.mark.gpu

CUTS = [(0, 1.0), (0, 0.9), (20, 1.0), (20, 0.9), (20, 0.3), (290, 0.9), (1, 0.5)]


def drawn(odla, x, temperatures, seed):
    rng = np.random.default_rng(seed)
    rows = [(t, k, p, u) for t in temperatures for k, p in CUTS for u in (0.02, 0.5, 0.97)]
    t, k, p, u = (np.array(a) for a in zip(*rows))
    logits = np.stack([np.asarray(x, np.float32)[rng.permutation(len(x))] for _ in rows])
    got, want = run_sample(odla, "fp32", logits, {"temperature": t, "top_k": k, "top_p": p, "uniform": u})
    assert np.array_equal(got, want), [(rows[i], int(g), int(w)) for i, (g, w) in enumerate(zip(got, want)) if g != w]
    return want


@pytest.mark.parametrize("v", [300, 5000])
def test_logits_whose_difference_is_beyond_fp32(odla, v):
    """3e38 and -3e38: their difference is infinite, their weights at a temperature of 1e38 or infinity are not 0."""
    announce("sampling from %d logits near the ends of fp32" % v)
    x = np.where(np.arange(v) % 3 == 0, 3e38, -3e38)
    x[1::7] = np.linspace(-1e38, 1e38, len(x[1::7]))
    want = drawn(odla, x, [np.inf, 1e38, 3e38, 1.0], v)
    assert len(set(want.tolist())) > 10


@pytest.mark.parametrize("v", [300, 5000])
def test_temperatures_whose_inverse_is_beyond_fp32(odla, v):
    """Subnormal temperatures over subnormal logits: log2(e) / T is infinite, (max - l) / T is not."""
    announce("sampling from %d subnormal logits" % v)
    t = np.float32(2.0 ** -140)
    x = -np.abs(np.random.default_rng(3).integers(0, 40, v)) * 2.0 ** -142
    want = drawn(odla, x, [float(t), float(t) * 16, 1e-37], v + 1)
    assert len(set(want.tolist())) > 10
