"""64-bit references of the operators of a token step, and the error bounds that their types give.

Tolerances: a result rounded to a type with machine epsilon `eps` (torch.finfo) is off by at most eps / 2 of its
value.  Sums of n fp32 products kept in 32 bits are off by at most n * 2^-23 times the sum of the absolute
products, in any order (2^-24 for each addition, doubled because the matrix instructions may truncate).
"""
import math

import numpy as np

BLOCK = 128
EPS = {"fp32": 2.0 ** -23, "fp16": 2.0 ** -10, "bf16": 2.0 ** -7}
LEAST = {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}   # smallest subnormal: what a rounding near zero is off by at most
UNIT = 2.0 ** -23


def blocks(n):
    return -(-n // BLOCK)


# ------------------------------------------------------------------- types --
def e4m3_table():
    b = np.arange(256)
    s, e, m = b >> 7, (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(float) - 10))
    v[(b & 127) == 127] = np.nan
    return np.where(s == 1, -v, v)


_TABLE = e4m3_table()


def e4m3_decode(bits):
    return _TABLE[np.asarray(bits)]


def e4m3_encode(x):
    """Bit patterns of the nearest values, ties to even, for |x| < 464; NaN gives 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isnan(x), 0.0, x))
    e = np.clip(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6, None)
    e = np.where(np.ldexp(1.0, (e + 1).astype(int)) <= a, e + 1, np.where(np.ldexp(1.0, e.astype(int)) > a, np.maximum(e - 1, -6), e))
    n = np.rint(a / np.ldexp(1.0, (e - 3).astype(int)))          # 8 .. 16, or 0 .. 8 below 2^-6
    up = n == 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    assert np.all(n * np.ldexp(1.0, (e - 3).astype(int)) <= 448), "beyond the type"
    bits = np.where(n < 8, n, ((e + 7) * 8) + (n - 8)).astype(np.int64)
    bits = np.where(np.isnan(x), 127, bits)
    return (bits | np.where(np.signbit(x) & ~np.isnan(x), 128, 0)).astype(np.uint8)


def to_bits(x, kind):
    """fp64 -> array that a HipBuilder argument of this type takes (rounded to nearest even)."""
    x = np.asarray(x)
    if kind == "fp32":
        return x.astype(np.float32)
    if kind == "fp16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = np.ascontiguousarray(x.astype(np.float32)).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def values(bits, kind):
    """What the array of to_bits stands for, in 64 bits."""
    if kind == "bf16":
        return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(bits).astype(np.float64)


# -------------------------------------------------------------- quantisation --
def quantize_rows(x):
    """(bit patterns, scales) of odla_hip_BlockQuantize in the 32-bit steps that the header names: exact."""
    x = np.asarray(x, np.float32)
    k = x.shape[-1]
    pad = np.zeros(x.shape[:-1] + (blocks(k) * BLOCK,), np.float32)
    pad[..., :k] = x
    b = pad.reshape(x.shape[:-1] + (-1, BLOCK))
    with np.errstate(invalid="ignore", over="ignore"):
        most = np.fmax.reduce(np.abs(b), axis=-1, initial=np.float32(0))
        scale = np.maximum(most / np.float32(448), np.float32(2.0 ** -126))
        q = e4m3_encode(b / scale[..., None])
    return q.reshape(pad.shape)[..., :k], scale


def row_values(q, scale):
    k = q.shape[-1]
    return e4m3_decode(q) * np.repeat(scale.astype(np.float64), BLOCK, axis=-1)[..., :k]


def quantize_squares(w):
    """(bit patterns, scales) for blocks of 128 x 128 of the last two dimensions."""
    r, k = w.shape[-2:]
    pad = np.zeros(w.shape[:-2] + (blocks(r) * BLOCK, blocks(k) * BLOCK))
    pad[..., :r, :k] = w
    b = pad.reshape(w.shape[:-2] + (blocks(r), BLOCK, blocks(k), BLOCK))
    scale = np.maximum(np.abs(b).max(axis=(-3, -1)) / 448.0, 2.0 ** -126).astype(np.float32)
    q = e4m3_encode(np.clip(b / scale[..., :, None, :, None].astype(np.float64), -448, 448))
    return np.ascontiguousarray(q.reshape(pad.shape)[..., :r, :k]), scale


def square_values(q, scale):
    r, k = q.shape[-2:]
    s = np.repeat(np.repeat(scale.astype(np.float64), BLOCK, axis=-2), BLOCK, axis=-1)[..., :r, :k]
    return e4m3_decode(q) * s


# ------------------------------------------------------------------- product --
def block_gemm(a, sa, b, sb, kind):
    """(result, bound) of odla_hip_BlockGemm."""
    av, bv = row_values(a, sa), square_values(b, sb)
    y = av @ bv.T
    terms = BLOCK + blocks(a.shape[-1]) + 3        # of a block, the blocks, the two scales and the last product
    off = terms * UNIT * (np.abs(av) @ np.abs(bv).T)
    if kind != "fp32":
        # 8-bit matrix instructions (more than 16 rows): of eight neighbouring products all but the largest lose up to 2^-13 of it
        for k in range(0, a.shape[-1], 8):
            off = off + 7 * 2.0 ** -13 * np.max([np.abs(av[..., j, None] * bv[:, j]) for j in range(k, min(k + 8, a.shape[-1]))], axis=0)
    return y, off + EPS[kind] / 2 * (np.abs(y) + off) + LEAST[kind]


# ------------------------------------------------------------------- experts --
def experts(x, router, gate_up, down, top_k, renormalize, scaling, kind, eight_bit=False):
    """(result, bound) of odla_hip_MixtureOfExperts on 64-bit values of its operands."""
    t, h = x.shape
    e, i = down.shape[0], down.shape[2]
    logits = x @ router.T
    off_l = (h + 2) * UNIT * (np.abs(x) @ np.abs(router).T)          # of a logit
    y, bound = np.zeros((t, h)), np.zeros((t, h))
    for r in range(t):
        order = np.lexsort((np.arange(e), -logits[r]))
        chosen = order[:top_k]
        if top_k < e:    # the choice must not hang on the last bits
            assert logits[r, order[top_k - 1]] - logits[r, order[top_k]] > 4 * off_l[r].max(), "a choice too close to call"
        w = np.exp(logits[r] - logits[r].max())
        share = w[chosen] / (w[chosen].sum() if renormalize else w.sum()) * scaling
        # exponentials: the logits' error, an fp32 argument, two units of expf; sums of up to E of them; quotient and scaling
        off_w = 2 * off_l[r].max() + 2 * UNIT * (np.ptp(logits[r]) + 2) + (e + 4) * UNIT
        for j, s in zip(chosen, share):
            extra = 4 if eight_bit else 0                              # block sums and their scales
            gate, up = gate_up[j, :i] @ x[r], gate_up[j, i:] @ x[r]
            off_g = (h + extra) * UNIT * (np.abs(gate_up[j, :i]) @ np.abs(x[r]))
            off_u = (h + extra) * UNIT * (np.abs(gate_up[j, i:]) @ np.abs(x[r]))
            silu = gate / (1 + np.exp(-gate))
            hidden = silu * up
            # the derivative of silu is at most 1.1; expf, sum, quotient and product take 8 units; then the rounding
            off_h = 1.1 * off_g * np.abs(up) + np.abs(silu) * off_u + 1.1 * off_g * off_u + 8 * UNIT * np.abs(hidden)
            off_h = off_h + EPS[kind] / 2 * (np.abs(hidden) + off_h) + LEAST[kind]
            y[r] += s * (down[j] @ hidden)
            a = np.abs(down[j])
            off = a @ off_h + (i + extra) * UNIT * (a @ (np.abs(hidden) + off_h))
            bound[r] += abs(s) * (off + (off_w + (top_k + 4) * UNIT) * (a @ (np.abs(hidden) + off_h)))
    return y, bound + EPS[kind] / 2 * (np.abs(y) + bound) + LEAST[kind]


# -------------------------------------------------------------------- sampling --
def sample_row(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.0):
    """The token of odla_hip_Sample, with weights as the whole numbers that the header names."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    if not l.max() > -np.inf:
        return -1
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(l == l.max(), 1.0, np.exp((l - l.max()) / float(temperature)))
    w = np.where(np.isnan(w), 0.0, w)
    f = [int(v) for v in np.rint(w * 2.0 ** 44)]
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        whole, run, n = sum(f[i] for i in order), 0, 0
        need = max(1, math.ceil(float(top_p) * float(whole)))
        while n < len(order) and (n == 0 or run < need):
            run += f[order[n]]
            n += 1
        order = order[:n]
    kept = sorted(int(i) for n, i in enumerate(order) if n == 0 or not w[i] < min_p)
    whole = sum(f[i] for i in kept)
    target = min(max(float(uniform), 0.0) * float(whole), whole - 1) if uniform == uniform else 0
    run = 0
    for i in kept:
        run += f[i]
        if run > target:
            return i
    raise AssertionError("nothing drawn")
