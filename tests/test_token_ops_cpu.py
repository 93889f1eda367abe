"""Operators of a token step without a GPU: result shapes, refusals, lowering, stored computations and the references
that the GPU tests compare with."""
import ctypes
import struct

import numpy as np
import pytest

import token_ops_ref as R


@pytest.fixture
def b(odla):
    hb = odla.HipBuilder()
    hb.L.odla_SetLogLevel(0)
    yield hb
    hb.L.odla_SetLogLevel(2)
    hb.destroy()


def f8(odla, b, name, shape):
    return b.arg(name, shape, odla.FLOAT8_E4M3)


def test_the_8_bit_code():
    v = R.e4m3_decode(np.arange(256))
    assert v[0x7e] == 448 and v[1] == 2.0 ** -9 and np.isnan(v[0x7f]) and np.isnan(v[0xff]) and np.isnan(v).sum() == 2
    fine = ~np.isnan(v)
    assert np.array_equal(R.e4m3_encode(v[fine]), np.arange(256)[fine])
    mid = (v[:0x7e] + v[1:0x7f]) / 2                      # ties go to the even pattern
    assert np.all(R.e4m3_encode(mid) % 2 == 0)
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).uniform(-448, 448, 5000) * 10.0 ** np.random.default_rng(1).integers(-5, 1, 5000)
    t = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.e4m3_encode(x.astype(np.float32)), t)


def test_shapes(odla, b):
    q, s = b.block_quantize(b.arg("x", (2, 3, 300), odla.BFLOAT16), names=("q", "s"))
    assert b.shape_of(q) == ((2, 3, 300), np.uint8) and b.shape_of(s) == ((2, 3, 3), np.float32)
    y = b.block_gemm(q, s, f8(odla, b, "w", (130, 300)), b.arg("ws", (2, 3)), odla.BFLOAT16)
    assert b.shape_of(y) == ((2, 3, 130), np.uint16)
    m = b.mixture_of_experts(b.arg("t", (4, 64)), b.arg("r", (6, 64)), b.arg("gu", (6, 40, 64)), b.arg("d", (6, 64, 20)), 2)
    assert b.shape_of(m) == ((4, 64), np.float32)
    t = b.sample(b.arg("l", (4, 5, 99), np.float16), b.arg("u", (4, 5)), temperature=b.arg("te", (1,)))
    assert b.shape_of(t) == ((4, 5), np.int32)
    assert b.shape_of(b.sample(b.arg("l1", (99,)), b.arg("u1", (1,)))) == ((1,), np.int32)


def test_refusals_of_the_quantisation(odla, b):
    for v in (b.arg("i", (3, 4), np.int32), f8(odla, b, "q", (3, 4))):
        with pytest.raises(odla.OdlaError):
            b.block_quantize(v)
    assert b.L.odla_hip_BlockQuantize(None, odla.ValueIds()).size == 0
    with pytest.raises(odla.OdlaError):
        b.block_quantize(b.arg("wide", (1, (1 << 24) + 1)))


def test_refusals_of_the_product(odla, b):
    a, sa = f8(odla, b, "a", (5, 200)), b.arg("sa", (5, 2))
    w, sw = f8(odla, b, "w", (130, 200)), b.arg("sw", (2, 2))
    b.block_gemm(a, sa, w, sw)
    bad = [(None, sa, w, sw, np.float32), (a, None, w, sw, np.float32), (a, sa, None, sw, np.float32), (a, sa, w, None, np.float32),
           (b.arg("af", (5, 200)), sa, w, sw, np.float32), (a, sa, b.arg("wf", (130, 200)), sw, np.float32),
           (a, b.arg("s1", (5, 1)), w, sw, np.float32), (a, b.arg("s2", (5, 2), np.float16), w, sw, np.float32),
           (a, sa, w, b.arg("s3", (1, 2)), np.float32), (a, sa, w, b.arg("s4", (130, 2)), np.float32),
           (a, sa, f8(odla, b, "w2", (130, 201)), sw, np.float32), (a, sa, f8(odla, b, "w3", (1, 130, 200)), sw, np.float32),
           (a, sa, w, sw, np.int32), (a, sa, w, sw, odla.FLOAT8_E4M3)]
    for args in bad:
        with pytest.raises(odla.OdlaError):
            b.block_gemm(*args)


def test_refusals_of_the_experts(odla, b):
    def args(**kw):
        shapes = {"x": (4, 64), "r": (6, 64), "gu": (6, 40, 64), "d": (6, 64, 20)}
        types = {n: np.float32 for n in shapes}
        shapes.update({n: v for n, v in kw.items() if n in shapes and isinstance(v, tuple)})
        types.update({n[:-1]: v for n, v in kw.items() if n.endswith("_")})
        return [b.arg(None, shapes[n], types[n]) for n in ("x", "r", "gu", "d")]

    b.mixture_of_experts(*args(), 2)
    for kw in ({"x": (4, 63)}, {"x": (513, 64)}, {"r": (5, 64)}, {"r": (6, 1, 64)}, {"gu": (6, 41, 64)}, {"gu": (6, 40, 63)}, {"d": (6, 63, 20)},
               {"d": (6, 64, 21)}, {"d": (6, 64 * 20)}, {"x_": np.float16}, {"r_": np.float16}, {"gu_": np.float16}, {"d_": odla.FLOAT8_E4M3},
               {"x_": np.int32, "r_": np.int32, "gu_": np.int32, "d_": np.int32}, {"gu_": odla.FLOAT8_E4M3, "d_": odla.FLOAT8_E4M3}):
        with pytest.raises(odla.OdlaError):
            b.mixture_of_experts(*args(**kw), 2)
    for k in (0, 7, 33):
        with pytest.raises(odla.OdlaError):
            b.mixture_of_experts(*args(), k)
    with pytest.raises(odla.OdlaError):
        b.mixture_of_experts(*args(), 2, gate_up_scale=b.arg("g", (6, 1, 1)))
    e8 = {"gu_": odla.FLOAT8_E4M3, "d_": odla.FLOAT8_E4M3}
    b.mixture_of_experts(*args(**e8), 2, b.arg("g1", (6, 1, 1)), b.arg("d1", (6, 1, 1)))
    for g, d in (((6, 1, 1), (6, 1, 2)), ((6, 2, 1), (6, 1, 1)), ((1, 1), (6, 1, 1))):
        with pytest.raises(odla.OdlaError):
            b.mixture_of_experts(*args(**e8), 2, b.arg(None, g), b.arg(None, d))
    big = [b.arg(None, s) for s in ((1, 8), (1025, 8), (1025, 4, 8), (1025, 8, 2))]
    with pytest.raises(odla.OdlaError):
        b.mixture_of_experts(*big, 2)
    many = [b.arg(None, s) for s in ((1, 8), (64, 8), (64, 4, 8), (64, 8, 2))]
    b.mixture_of_experts(*many, 32)
    with pytest.raises(odla.OdlaError):
        b.mixture_of_experts(*many, 33)


@pytest.mark.parametrize("tokens,hidden,inner,top_k", [(512, 1 << 21, 4, 1), (512, 4, 1 << 16, 32), (64, 4, 1 << 23, 2)])
def test_refusal_of_experts_behind_32_bit_offsets(odla, b, tokens, hidden, inner, top_k):
    def layer(t):
        b.mixture_of_experts(b.arg(None, (t, hidden)), b.arg(None, (64, hidden)), b.arg(None, (64, 2 * inner, hidden)),
                             b.arg(None, (64, hidden, inner)), top_k)
    layer(tokens - 1)
    with pytest.raises(odla.OdlaError):
        layer(tokens)


def test_refusals_of_the_sampling(odla, b):
    l, u = b.arg("l", (4, 100)), b.arg("u", (4,))
    b.sample(l, u)
    for args, kw in (((b.arg("li", (4, 100), np.int32), u), {}), ((l, b.arg("u3", (3,))), {}), ((l, b.arg("uh", (4,), np.float16)), {}),
                     ((l, None), {}), ((None, u), {}), ((l, u), {"top_k": b.arg("kf", (4,))}), ((l, u), {"top_k": b.arg("kl", (4,), np.int64)}),
                     ((l, u), {"top_p": b.arg("pi", (4,), np.int32)}), ((l, u), {"min_p": b.arg("m5", (5,))}),
                     ((l, u), {"temperature": b.arg("t100", (100,))}), ((b.arg("long", (4, (1 << 19) + 1)), u), {})):
        with pytest.raises(odla.OdlaError):
            b.sample(*args, **kw)


def test_other_operators_refuse_8_bit_values(odla, b):
    q, r = f8(odla, b, "q", (4, 6)), f8(odla, b, "r", (1, 4, 6, 6))
    for op in (lambda: b.relu(q), lambda: b.add(q, q), lambda: b.equal(q, q), lambda: b.cast(q, np.float32), lambda: b.softmax(q),
               lambda: b.reduce_sum(q, [1]), lambda: b.maxpool(r, (2, 2), (1, 1), (0, 0, 0, 0)), lambda: b.gemm(q, b.arg("w", (6, 2))),
               lambda: b.topk(q, 2, 1), lambda: b.tile(q, (2, 1)), lambda: b.pad(q, (1, 0), (0, 0)), lambda: b.argmax(q, 1)):
        with pytest.raises(odla.OdlaError):
            op()
    with pytest.raises(odla.OdlaError):      # and none gives them
        b._ret(b.L.odla_Cast(b.arg("x", (4, 6)), odla.ODLA_HIP_FLOAT8_E4M3, None), "odla_Cast")
    for v, shape in ((b.reshape(q, (24,)), (24,)), (b.transpose(q, (1, 0)), (6, 4)), (b.slice(q, (0, 1), (4, 3)), (4, 2)),
                     (b.concat([q, q], 0), (8, 6)), (b.gather(q, b.const("i", np.array([1], np.int32))), (1, 6))):
        assert b.shape_of(v)[0] == shape


def record_step(odla, b, batch):
    x = b.arg("x", (batch, 8), odla.BFLOAT16)
    y = b.mixture_of_experts(x, b.const("r", np.zeros((3, 8), np.uint16), odla.BFLOAT16),
                             b.const("gu", np.zeros((3, 8, 8), np.uint8), odla.FLOAT8_E4M3), b.const("d", np.zeros((3, 8, 4), np.uint8), odla.FLOAT8_E4M3),
                             2, b.const("gs", np.ones((3, 1, 1), np.float32)), b.const("ds", np.ones((3, 1, 1), np.float32)), name="moe")
    q, s = b.block_quantize(y, names=("q", "s"))
    l = b.block_gemm(q, s, b.const("w", np.zeros((9, 8), np.uint8), odla.FLOAT8_E4M3), b.const("ws", np.ones((1, 1), np.float32)), name="l")
    b.output(b.sample(l, b.arg("u", (batch,)), top_k=b.const("k", np.array([5], np.int32)), name="token"), "token")


@pytest.mark.parametrize("mode", [{}, {"fp16": True}, {"bf16": True}, {"bf16": "accuracy"}])
def test_lowering(odla, mode):
    hb = odla.HipBuilder(**mode)
    try:
        record_step(odla, hb, 4)
        s = hb.plan_summary()
        assert s["launches"] >= 6 and s["arena_bytes"] > 0
    finally:
        hb.destroy()


def stored_step(odla, path):
    hb = odla.HipBuilder()
    try:
        record_step(odla, hb, 4)
        loc, keep = odla.path_location(path)
        assert hb.L.odla_StoreComputation(loc, hb.comp) == 0
    finally:
        hb.destroy()
    return open(path, "rb").read()


def load(odla, data):
    L = odla.load_library()
    loc, keep = odla.memory_location(data)
    comp = ctypes.c_void_p()
    L.odla_SetLogLevel(0)
    st = L.odla_LoadComputation(loc, ctypes.byref(comp))
    L.odla_SetLogLevel(2)
    if st == 0:
        ps = odla.PlanSummary()
        assert L.odla_hip_PlanSummary(comp, ctypes.byref(ps)) == 0
        assert L.odla_DestroyComputation(comp) == 0
    return st


def rehashed(data):
    h = 1469598103934665603
    for c in data:
        h = ((h ^ c) * 0x100000001b3) & (2 ** 64 - 1)
    return data + struct.pack("<Q", h)


def test_stored_and_loaded(odla, tmp_path):
    data = stored_step(odla, str(tmp_path / "step.odla"))
    assert load(odla, data) == 0
    assert rehashed(data[:-8]) == data        # (the hash below is the file's own)


def test_damaged_attributes_are_rejected(odla, tmp_path):
    """Numbers anywhere in a stored step replaced by others: it loads as something the planner accepts, or is refused."""
    data = stored_step(odla, str(tmp_path / "step.odla"))[:-8]
    L = odla.load_library()
    rejected = 0
    L.odla_SetLogLevel(0)
    for at in range(8, len(data) - 8, 3):
        for new in (-1, 3, 31, 1 << 40):
            bad = bytearray(data)
            struct.pack_into("<q", bad, at, new)
            loc, keep = odla.memory_location(rehashed(bytes(bad)))
            comp = ctypes.c_void_p()
            if L.odla_LoadComputation(loc, ctypes.byref(comp)) == 0:
                ps = odla.PlanSummary()
                L.odla_hip_PlanSummary(comp, ctypes.byref(ps))
                L.odla_DestroyComputation(comp)
            else:
                rejected += 1
    L.odla_SetLogLevel(2)
    assert rejected > 50


def test_reference_of_the_sampling():
    l = np.log([0.5, 0.25, 0.125, 0.125])
    assert [R.sample_row(l, uniform=u) for u in (0.0, 0.49, 0.51, 0.76, 0.9)] == [0, 0, 1, 2, 3]
    assert R.sample_row(l, top_k=2, uniform=0.999) == 1 and R.sample_row(l, top_p=0.5, uniform=0.999) == 0
    assert R.sample_row(l, min_p=0.3, uniform=0.999) == 1 and R.sample_row(l[::-1], temperature=0.0) == 3
    assert R.sample_row([-np.inf, np.nan]) == -1 and R.sample_row([2.0, 2.0, 2.0], top_k=2, uniform=0.99) == 1
