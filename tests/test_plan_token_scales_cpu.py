"""Lowering of scales and sampling parameters behind moving operators, without a GPU."""
import numpy as np
import pytest

import token_scale_graphs as G


def launches(odla, build, **mode):
    hb = odla.HipBuilder(**mode)
    try:
        build(hb)
        return hb.plan_summary()["launches"]
    finally:
        hb.destroy()


@pytest.mark.parametrize("mode", [{"fp16": True}, {"bf16": True}, {"bf16": "accuracy"}])
@pytest.mark.parametrize("move", list(G.MOVES))
def test_moved_scales_are_not_converted(odla, move, mode):
    """The precision modes store FLOAT32 values in 16 bits; scales on the way to a product are launched as in fp32 mode."""
    x, w, ws = G.moved_operands()
    build = G.moved_product(odla, move, w, ws)
    assert launches(odla, build, **mode) == launches(odla, build)


@pytest.mark.parametrize("mode", [{"fp16": True}, {"bf16": True}])
def test_moved_parameters_are_not_converted(odla, mode):
    def build(b):
        p = b.arg("p", (3, 4))
        part = lambda i: b.reshape(b.slice(p, (i, 0), (i + 1, 4)), (4,))
        b.output(b.sample(b.arg("l", (4, 50), np.float16), part(0), temperature=part(1), top_p=part(2), name="t"), "t")

    def tiled(b):
        one = b.arg("p", (1,))
        b.output(b.sample(b.arg("l", (4, 50), np.float16), b.tile(one, (4,)), min_p=b.broadcast_to(one, (4,)), name="t"), "t")
    assert launches(odla, build, **mode) == launches(odla, build)
    assert launches(odla, tiled, **mode) == launches(odla, tiled)
