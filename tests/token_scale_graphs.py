"""Graphs in which scales and sampling parameters pass moving operators on the way to their readers."""
import numpy as np

import token_ops_ref as R

# one graph per moving operator: rows [6, 300] quantised, values and scales moved alike, and multiplied
MOVES = {
    "none": lambda b, v, w: v,
    "reshape": lambda b, v, w: b.reshape(b.reshape(v, (2, 3, w)), (6, w)),
    "slice": lambda b, v, w: b.slice(v, (1, 0), (6, w), (2, 1)),
    "transpose": lambda b, v, w: b.transpose(b.transpose(v, (1, 0)), (1, 0)),
    "concat": lambda b, v, w: b.concat([v, v], 0),
    "gather": lambda b, v, w: b.gather(v, b.const(None, np.array([5, 0, 3, 3], np.int32)), 0),
    "channels": lambda b, v, w: b.reshape(b.concat([b.reshape(v, (2, 3, 1, w)), b.reshape(v, (2, 3, 1, w))], 1), (12, w)),
}
ROWS = {
    "none": lambda a: a,
    "reshape": lambda a: a,
    "slice": lambda a: a[1:6:2],
    "transpose": lambda a: a,
    "concat": lambda a: np.concatenate([a, a]),
    "gather": lambda a: a[[5, 0, 3, 3]],
    "channels": lambda a: np.concatenate([a.reshape(2, 3, -1)] * 2, 1).reshape(12, -1),
}


def moved_product(odla, move, w, ws, outputs=False):
    def build(b):
        q, s = b.block_quantize(b.arg("x", (6, 300), np.float16), names=("q", "s"))
        mq, ms = MOVES[move](b, q, 300), MOVES[move](b, s, 3)
        y = b.block_gemm(mq, ms, b.const("w", w, odla.FLOAT8_E4M3), b.reshape(b.const("ws", ws.reshape(-1)), ws.shape), np.float16, name="y")
        b.output(y, "y")
        if outputs:
            b.output(ms, "ms")
            b.output(b.mul(ms, ms, name="twice"), "twice")       # (a reader of another kind)
    return build


def moved_operands():
    rng = np.random.default_rng(41)
    x = rng.standard_normal((6, 300)).astype(np.float16)
    w, ws = R.quantize_squares(rng.standard_normal((200, 300)))
    return x, w, ws
