"""Norm, attention over a paged cache and log probabilities without a GPU: result shapes, refusals, lowering and stored
computations."""
import ctypes
import struct

import numpy as np
import pytest


@pytest.fixture
def b(odla):
    hb = odla.HipBuilder()
    hb.L.odla_SetLogLevel(0)
    yield hb
    hb.L.odla_SetLogLevel(2)
    hb.destroy()


def refused(odla, call):
    with pytest.raises(odla.OdlaError):
        call()


def attention(odla, b, kind=np.float32, t=6, hq=4, h=2, d=16, pages=8, page=4, seqs=3, width=5, fresh=True, starts=True, flat=False, **kw):
    q = b.arg("q", (t, hq * d) if flat else (t, hq, d), kind)
    k, v = (b.arg(n, (t, h * d) if flat else (t, h, d), kind) if fresh else None for n in "kv")
    return b.paged_attention(q, k, v, b.arg("kc", (pages, page, h, d), kind), b.arg("vc", (pages, page, h, d), kind), b.arg("pt", (seqs, width), np.int32),
                             b.arg("n", (seqs,), np.int32), b.arg("s", (seqs + 1,), np.int32) if starts else None, name="y", **kw)


def test_shapes(odla, b):
    x, r = b.arg("x", (2, 3, 300), odla.BFLOAT16), b.arg("r", (2, 3, 300), odla.BFLOAT16)
    shapes = lambda got: [b.shape_of(v) for v in got]
    assert shapes(b.rms_norm(x)) == [((2, 3, 300), np.uint16)]
    assert shapes(b.rms_norm(x, residual=r)) == [((2, 3, 300), np.uint16)] * 2
    assert shapes(b.rms_norm(x, b.arg("w", (300,)), dtype=odla.FLOAT8_E4M3)) == [((2, 3, 300), np.uint8), ((2, 3, 3), np.float32)]
    assert shapes(b.rms_norm(x, b.arg("w2", (300,), odla.BFLOAT16), r, dtype=odla.FLOAT8_E4M3)) == [
        ((2, 3, 300), np.uint8), ((2, 3, 3), np.float32), ((2, 3, 300), np.uint16)]
    l = b.arg("l", (4, 5, 99), np.float16)
    assert shapes(b.log_probs(l, b.arg("t", (4, 5), np.int32))) == [((4, 5), np.float32)] * 2
    assert shapes(b.log_probs(l, b.arg("t7", (4, 5, 7), np.int32), 3)) == [((4, 5, 7), np.float32), ((4, 5), np.float32), ((4, 5, 3), np.float32), ((4, 5, 3), np.int32)]
    assert shapes(b.log_probs(b.arg("l1", (99,)), b.arg("t1", (1,), np.int32), 2)) == [((1,), np.float32), ((1,), np.float32), ((2,), np.float32), ((2,), np.int32)]
    assert b.shape_of(attention(odla, b)) == ((6, 4, 16), np.float32)


def test_attention_takes_flat_rows_and_equal_sequences(odla, b):
    assert b.shape_of(attention(odla, b, np.float16, flat=True, starts=False, window=3)) == ((6, 64), np.float16)


def test_refusals_of_the_norm(odla, b):
    x = b.arg("x", (3, 40), np.float16)
    refused(odla, lambda: b.rms_norm(b.arg("i", (3, 40), np.int32)))
    refused(odla, lambda: b.rms_norm(b.arg("q", (3, 40), odla.FLOAT8_E4M3)))
    refused(odla, lambda: b.rms_norm(x, b.arg("w", (39,))))
    refused(odla, lambda: b.rms_norm(x, b.arg("w2", (40,), odla.BFLOAT16)))
    refused(odla, lambda: b.rms_norm(x, residual=b.arg("r", (3, 40))))
    refused(odla, lambda: b.rms_norm(x, residual=b.arg("r2", (4, 40), np.float16)))
    refused(odla, lambda: b.rms_norm(x, dtype=np.float32))
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(odla, lambda: b.rms_norm(x, epsilon=eps))
    refused(odla, lambda: b.rms_norm(b.arg("wide", (1, (1 << 24) + 1))))
    assert b.L.odla_hip_RmsNorm(None, None, None, 1e-6, odla.ODLA_FLOAT32, odla.ValueIds()).size == 0
    other = odla.HipBuilder()
    refused(odla, lambda: b.rms_norm(x, other.arg("w", (40,))))
    other.destroy()


@pytest.mark.parametrize("kw", [dict(d=12), dict(d=264), dict(hq=3), dict(seqs=2, t=5, starts=False), dict(kind=np.int32), dict(page=1 << 29, width=3),
                                dict(pages=1 << 16, page=1 << 15), dict(seqs=65537, t=65537), dict(scale=float("nan")), dict(scale=float("inf"))])
def test_refusals_of_the_attention(odla, b, kw):
    refused(odla, lambda: attention(odla, b, **kw))


def test_refused_operands_of_the_attention(odla, b):
    kind = odla.BFLOAT16
    q, k, v = b.arg("q", (6, 4, 16), kind), b.arg("k", (6, 2, 16), kind), b.arg("v", (6, 2, 16), kind)
    kc, vc = b.arg("kc", (8, 4, 2, 16), kind), b.arg("vc", (8, 4, 2, 16), kind)
    pt, n, s = b.arg("pt", (3, 5), np.int32), b.arg("n", (3,), np.int32), b.arg("s", (4,), np.int32)
    b.paged_attention(q, k, v, kc, vc, pt, n, s)
    b.paged_attention(q, None, None, kc, vc, pt, n, s)
    tries = [(q, k, None, kc, vc, pt, n, s), (q, None, v, kc, vc, pt, n, s), (q, k, v, kc, kc, pt, n, s), (q, k, v, kc, b.arg("vc2", (8, 4, 2, 24), kind), pt, n, s),
             (q, k, v, b.const("c", np.zeros((8, 4, 2, 16), np.uint16), kind), vc, pt, n, s), (q, k, v, kc, b.reshape(vc, (8, 4, 2, 16)), pt, n, s),
             (q, b.arg("k3", (5, 2, 16), kind), v, kc, vc, pt, n, s), (q, b.arg("k4", (6, 2, 16), np.float16), v, kc, vc, pt, n, s),
             (b.arg("q2", (6, 4, 16)), k, v, kc, vc, pt, n, s), (b.arg("q3", (6, 4, 8), kind), k, v, kc, vc, pt, n, s), (b.arg("q4", (6, 2, 2, 16), kind), k, v, kc, vc, pt, n, s),
             (q, k, v, kc, vc, b.arg("pt2", (15,), np.int32), n, s), (q, k, v, kc, vc, b.arg("pt3", (3, 5), np.int64), n, s),
             (q, k, v, kc, vc, pt, b.arg("n2", (2,), np.int32), s), (q, k, v, kc, vc, pt, n, b.arg("s2", (3,), np.int32)), (q, k, v, kc, vc, pt, n, b.arg("s3", (4,)))]
    for ops in tries:
        refused(odla, lambda: b.paged_attention(*ops[:7], starts=ops[7], scale=1.0))
    assert not b.L.odla_hip_PagedAttention(None, k, v, kc, vc, pt, n, s, 1.0, 0, None)
    assert not b.L.odla_hip_PagedAttention(q, k, v, None, vc, pt, n, s, 1.0, 0, None)
    assert not b.L.odla_hip_PagedAttention(q, k, v, kc, vc, None, n, s, 1.0, 0, None)
    assert not b.L.odla_hip_PagedAttention(q, k, v, kc, vc, pt, None, s, 1.0, 0, None)


def test_refusals_of_the_log_probabilities(odla, b):
    l, t = b.arg("l", (4, 99)), b.arg("t", (4,), np.int32)
    for top in (33, 100, -1 & 0xffffffff):
        refused(odla, lambda: b.log_probs(l, t, top))
    refused(odla, lambda: b.log_probs(b.arg("few", (4, 5)), t, 6))
    refused(odla, lambda: b.log_probs(l, b.arg("tf", (4,))))
    refused(odla, lambda: b.log_probs(l, b.arg("t3", (3,), np.int32)))
    refused(odla, lambda: b.log_probs(l, b.arg("t65", (4, 65), np.int32)))
    refused(odla, lambda: b.log_probs(b.arg("i", (4, 99), np.int32), t))
    refused(odla, lambda: b.log_probs(b.arg("wide", (4, 524289)), t))
    assert b.L.odla_hip_LogProbs(None, t, 0, odla.ValueIds()).size == 0


def test_a_cache_has_no_other_reader(odla, b):
    """A copy of a cache in another form would go stale when it is extended: refused when the computation is lowered."""
    b.output(attention(odla, b), "y")
    kc = b.args["kc"][0]
    assert b.plan_summary()["launches"] == 2
    b.output(b.slice(kc, (0, 0, 0, 0), (1, 4, 2, 16)), "part") if hasattr(b, "slice") else b.output(b.transpose(kc, (1, 0, 2, 3)), "part")
    refused(odla, b.plan_summary)


def test_a_cache_is_no_output(odla, b):
    b.output(attention(odla, b), "y")
    b.output(b.args["kc"][0], "kc_out")
    refused(odla, b.plan_summary)


def test_a_cache_takes_no_room(odla):
    """Caches are the caller's: the plan holds nothing of their size."""
    hb = odla.HipBuilder()
    hb.output(attention(odla, hb, odla.BFLOAT16, pages=1 << 14, page=64, h=8, hq=8, d=128), "y")
    assert hb.plan_summary()["arena_bytes"] < 64 << 20
    hb.destroy()


@pytest.mark.parametrize("mode", [{}, {"fp16": True}, {"bf16": True}, {"bf16": "accuracy"}])
def test_launches(odla, mode):
    """One launch a norm, whatever it gives; two an attention; one or two for log probabilities."""
    hb = odla.HipBuilder(**mode)
    got = hb.rms_norm(hb.arg("x", (7, 300), odla.BFLOAT16), hb.arg("w", (300,), odla.BFLOAT16), hb.arg("r", (7, 300), odla.BFLOAT16), dtype=odla.FLOAT8_E4M3)
    for v, n in zip(got, ("q", "scale", "sum")):
        hb.output(v, n)
    assert hb.plan_summary()["launches"] == 1
    hb.destroy()
    for v, launches in ((500, 1), (32768, 1), (32769, 2)):
        hb = odla.HipBuilder(**mode)
        for x, n in zip(hb.log_probs(hb.arg("l", (3, v), np.float16), hb.arg("t", (3,), np.int32), 4), ("lp", "e", "tl", "tt")):
            hb.output(x, n)
        assert hb.plan_summary()["launches"] == launches
        hb.destroy()
    hb = odla.HipBuilder(**mode)
    hb.output(attention(odla, hb, np.float16), "y")
    assert hb.plan_summary()["launches"] == 2
    hb.destroy()


def record(odla, b):
    x = b.arg("x", (6, 64), odla.BFLOAT16)
    q, s, z = b.rms_norm(x, b.const("w", np.ones(64, np.float32)), b.arg("r", (6, 64), odla.BFLOAT16), dtype=odla.FLOAT8_E4M3, names=("q", "scale", "sum"))
    y = attention(odla, b, odla.BFLOAT16, flat=True)
    for v, n in zip(b.log_probs(y, b.arg("t", (6,), np.int32), 5, names=("lp", "e", "tl", "tt")) + (q, s, z), ("lp", "e", "tl", "tt", "q", "scale", "sum")):
        b.output(v, n)


def load(odla, L, blob):
    comp = ctypes.c_void_p()
    loc, keep = odla.memory_location(bytes(blob))
    return L.odla_LoadComputation(loc, ctypes.byref(comp)), comp, keep


def fnv(data):
    h = 1469598103934665603
    for x in data:
        h = (h ^ x) * 1099511628211 & (1 << 64) - 1
    return h


def test_stored_and_loaded(odla, b, tmp_path):
    record(odla, b)
    want = b.plan_summary()
    path = str(tmp_path / "layer.odla")
    loc, keep = odla.path_location(path)
    assert b.L.odla_StoreComputation(loc, b.comp) == 0
    blob = open(path, "rb").read()
    status, comp, keep = load(odla, b.L, blob)
    assert status == 0
    ps = odla.PlanSummary()
    assert b.L.odla_hip_PlanSummary(comp, ctypes.byref(ps)) == 0
    assert ps.launches == want["launches"] and ps.arena_bytes == want["arena_bytes"]
    assert b.L.odla_DestroyComputation(comp) == 0


def test_damaged_files_are_refused(odla, b, tmp_path):
    """Every word of the nodes' records changed in turn, with a hash that fits: refused, or a computation that lowers or is
    refused then; never a crash."""
    record(odla, b)
    path = str(tmp_path / "layer.odla")
    loc, keep = odla.path_location(path)
    assert b.L.odla_StoreComputation(loc, b.comp) == 0
    blob = bytearray(open(path, "rb").read())
    refused_ones = 0
    for at in range(len(blob) - 8 - 8 * 160, len(blob) - 8, 8):
        for word in (-1, 1, 77, 1 << 40):
            bad = bytearray(blob)
            bad[at:at + 8] = struct.pack("<q", word)
            bad[-8:] = struct.pack("<Q", fnv(bad[:-8]))
            status, comp, keep = load(odla, b.L, bad)
            if status == 0:
                b.L.odla_hip_PlanSummary(comp, ctypes.byref(odla.PlanSummary()))
                b.L.odla_DestroyComputation(comp)
            else:
                refused_ones += 1
    assert refused_ones > 50


def test_dynamic_batch_is_recorded(odla):
    """Sequences as the batch: equal lengths, caches of their own size."""
    hb = odla.HipBuilder(max_batch=8)
    kind = odla.BFLOAT16
    x = hb.arg("x", (-1, 64), kind)
    y, z = hb.rms_norm(x, residual=hb.arg("r", (-1, 64), kind))
    a = hb.paged_attention(y, hb.arg("k", (-1, 32), kind), hb.arg("v", (-1, 32), kind), hb.arg("kc", (8, 4, 2, 16), kind), hb.arg("vc", (8, 4, 2, 16), kind),
                           hb.arg("pt", (-1, 5), np.int32), hb.arg("n", (-1,), np.int32))
    assert hb.shape_of(a) == ((8, 64), np.uint16)
    hb.output(hb.log_probs(a, hb.arg("t", (-1,), np.int32), 2)[0], "lp")
    assert hb.plan_summary()["launches"] == 4
    hb.destroy()


@pytest.mark.parametrize("mode,kind", [({"fp16": True}, "BFLOAT16"), ({"bf16": True}, np.float16)])
def test_weight_of_a_norm_whose_input_the_mode_does_not_store(odla, mode, kind):
    """A FLOAT32 weight beside an input in the other 16-bit type stays fp32: one launch, four bytes an element; beside one in the
    mode's type it takes two."""
    room = {}
    other = {"fp16": np.float16, "bf16": odla.BFLOAT16}[next(iter(mode))]
    for x_kind in (getattr(odla, kind) if isinstance(kind, str) else kind, other):
        for constant in (True, False):
            hb = odla.HipBuilder(**mode)
            w = hb.const("w", np.ones(3000, np.float32)) if constant else hb.arg("w", (3000,))
            hb.output(hb.rms_norm(hb.arg("x", (2, 3000), x_kind), w)[0], "y")
            room[x_kind is other, constant] = hb.plan_summary()
            hb.destroy()
    assert room[False, True]["launches"] == room[False, False]["launches"] == room[True, True]["launches"] == 1
    assert room[True, False]["launches"] == 2           # (the cast of an argument)
    assert room[False, True]["constant_bytes"] >= 4 * 3000 > room[True, True]["constant_bytes"] >= 2 * 3000


def test_calls_that_no_launch_has_room_for_are_refused(odla):
    """A launch has less than 2^32 lanes: both sides of where the operators' launches reach that."""
    hb = odla.HipBuilder()
    hb.L.odla_SetLogLevel(0)
    try:
        bf16, n = odla.BFLOAT16, [0]

        def arg(shape, kind=bf16):
            n[0] += 1
            return hb.arg("a%d" % n[0], shape, kind)

        for rows, k, fits in ((65535 * 128, 4096, True), (2 ** 22 - 1, 4097, True), (2 ** 22, 4097, False)):
            call = lambda: hb.rms_norm(arg((rows, k)))
            call() if fits else refused(odla, call)
        for rows, v, top, fits in ((65535 * 128, 8192, 1, True), (2 ** 22 - 1, 8193, 1, True), (2 ** 22, 8193, 1, False), (2 ** 22, 8193, 0, True),
                                   (2 ** 21 - 1, 32769, 1, True), (2 ** 21, 32769, 1, False)):
            call = lambda: hb.log_probs(arg((rows, v)), arg((rows,), np.int32), top)
            call() if fits else refused(odla, call)
        for seqs, heads, group, kind, fits in ((250, 65535, 1, bf16, True), (257, 65535, 1, bf16, False), (4000, 1000, 60, bf16, True), (4000, 1000, 70, np.float32, False)):
            rows = lambda: arg((seqs, heads * 8), kind)
            cache = lambda: arg((seqs, 1, heads, 8), kind)
            call = lambda: hb.paged_attention(arg((seqs, heads * group * 8), kind), rows(), rows(), cache(), cache(), arg((seqs, 1), np.int32), arg((seqs,), np.int32))
            call() if fits else refused(odla, call)
    finally:
        hb.L.odla_SetLogLevel(2)
        hb.destroy()
