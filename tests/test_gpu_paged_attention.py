"""odla_hip_PagedAttention against the formula in 64 bits: head layouts, lengths, page sizes, windows, odd operands; the
caches as they are afterwards; captured and replayed, stored, in the precision modes."""
import numpy as np
import pytest

import layer_ops_ref as L
import token_ops_ref as R
from test_gpu_token_ops import np_kind
from util import announce

pytestmark = pytest.mark.gpu

KINDS = ["fp32", "fp16", "bf16"]


class Case:
    """Operands of a call; garbage wherever no token of a sequence lies."""

    def __init__(self, kind, new, cached, heads=2, group=2, d=32, page=16, spare=2, seed=0, starts=True, fresh=True, tail=0, window=0, scale=None, junk=None):
        rng = np.random.default_rng(seed)
        self.kind, self.window, self.fresh = kind, window, fresh
        self.scale = d ** -0.5 if scale is None else scale
        new, cached = list(new), list(cached)
        b, t = len(new), sum(new) + tail
        owned = [-(-(n + c) // page) for n, c in zip(new, cached)]
        pages = max(1, sum(owned) + spare)
        order = rng.permutation(pages)
        self.table = np.full((b, max(owned + [1]) + 1), -1, np.int32)
        ends = np.cumsum([0] + owned)
        for i, n in enumerate(owned):
            self.table[i, :n] = order[ends[i]:ends[i] + n]
        bits = lambda *shape: R.to_bits(rng.standard_normal(shape), kind)
        self.q, self.k, self.v = bits(t, heads * group, d), bits(t, heads, d), bits(t, heads, d)
        self.kc, self.vc = bits(pages, page, heads, d), bits(pages, page, heads, d)
        self.cached = np.array(cached, np.int32)
        self.starts = np.cumsum([0] + new).astype(np.int32) if starts else None
        if not fresh:      # the new tokens lie in the caches already
            for i, (n, c) in enumerate(zip(new, cached)):
                for j in range(n):
                    at = (self.table[i, (c + j) // page], (c + j) % page)
                    self.kc[at], self.vc[at] = self.k[sum(new[:i]) + j], self.v[sum(new[:i]) + j]
        if junk is not None:   # places that no sequence owns
            mine = np.zeros((pages, page), bool)
            for i, (n, c) in enumerate(zip(new, cached)):
                for p in range(c + n):
                    mine[self.table[i, p // page], p % page] = True
            for cache in (self.kc, self.vc):
                cache[~mine] = R.to_bits(np.full(cache[~mine].shape, junk), kind)

    def record(self, odla, b, mode_kind=None):
        kind = np_kind(odla, mode_kind or self.kind)
        args = {"q": self.q, "k": self.k, "v": self.v, "kc": self.kc, "vc": self.vc}
        h = {n: b.arg(n, a.shape, kind) for n, a in args.items() if self.fresh or n not in "kv"}
        return b.paged_attention(h["q"], h.get("k"), h.get("v"), h["kc"], h["vc"], b.arg("pt", self.table.shape, np.int32), b.arg("n", self.cached.shape, np.int32),
                                 None if self.starts is None else b.arg("s", self.starts.shape, np.int32), self.scale, self.window, "y")

    def feeds(self, odla):
        f = {"q": self.q, "pt": self.table, "n": self.cached, "kc": odla.DeviceArray(self.kc), "vc": odla.DeviceArray(self.vc)}
        if self.fresh:
            f.update(k=self.k, v=self.v)
        if self.starts is not None:
            f["s"] = self.starts
        return f

    def written(self):
        """Both caches' bits afterwards: what no token is written to stays as it was."""
        kc, vc = self.kc.copy(), self.vc.copy()
        pages, page = kc.shape[:2]
        starts = np.arange(len(self.cached) + 1) * (len(self.q) // len(self.cached)) if self.starts is None else self.starts
        for i, row in enumerate(self.table):
            before = min(max(int(self.cached[i]), 0), len(row) * page)
            for j in range(starts[i], starts[i + 1]):
                place = before + j - starts[i]
                if self.fresh and place < len(row) * page and 0 <= row[place // page] < pages:
                    kc[row[place // page], place % page], vc[row[place // page], place % page] = self.k[j], self.v[j]
        return kc, vc

    def want(self):
        v = lambda a: R.values(a, self.kind)
        return L.paged_attention(v(self.q), v(self.k) if self.fresh else None, v(self.v), v(self.kc), v(self.vc), self.table, self.cached, self.starts,
                                 self.scale, self.window, self.kind)


def run(odla, c, repeats=1, **mode):
    """Result bits and both caches' bits; executed `repeats` times (the same tokens to the same places)."""
    b = odla.HipBuilder(**mode)
    feeds = c.feeds(odla)
    try:
        b.output(c.record(odla, b), "y")
        s = b.session()
        try:
            first = None
            for _ in range(repeats):
                y = s.run(feeds)["y"]
                assert first is None or np.array_equal(y, first)
                first = y
        finally:
            s.close()
        return y, feeds["kc"].get(), feeds["vc"].get()
    finally:
        feeds["kc"].close()
        feeds["vc"].close()
        b.destroy()


def check(odla, c, **kw):
    y, kc, vc = run(odla, c, **kw)
    want, bound, _, _ = c.want()
    kc_want, vc_want = c.written()
    assert np.array_equal(kc.view(np.uint8), kc_want.view(np.uint8)) and np.array_equal(vc.view(np.uint8), vc_want.view(np.uint8))
    have = R.values(y, c.kind)
    with np.errstate(invalid="ignore"):
        off = np.abs(have - want)
    assert np.all((off <= bound) | (have == want)), "%d of %d off, worst %g of its bound" % (np.sum(off > bound), off.size, np.nanmax(off / np.maximum(bound, 1e-300)))
    return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [8, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (1, 16), (3, 5), (2, 20)])
def test_heads(odla, kind, d, heads, group):
    announce("paged attention %s heads %d x %d of %d" % (kind, heads, group, d))
    check(odla, Case(kind, [1, 3, 1], [40, 0, 75], heads, group, d, seed=d + group))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 3, 16, 20, 64, 1000])
def test_pages(odla, kind, page):
    announce("paged attention %s pages of %d" % (kind, page))
    check(odla, Case(kind, [1, 9, 2, 1], [130, 33, 0, 64], page=page, seed=page, d=64))


LENGTHS = [([1], [0]), ([1], [1]), ([1], [31]), ([1], [32]), ([1], [4095]), ([2], [15]), ([16], [0]), ([17], [0]), ([33], [100]), ([64], [0]), ([65], [63]),
           ([129], [0]), ([300], [500]), ([1, 1, 1, 1], [5, 2000, 0, 300]), ([40, 1, 1, 7], [0, 900, 33, 256]), ([0, 5, 0, 0, 1, 0], [10, 20, 0, 700, 3, 0])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,cached", LENGTHS)
def test_lengths(odla, kind, new, cached):
    announce("paged attention %s new %s cached %s" % (kind, new, cached))
    check(odla, Case(kind, new, cached, 2, 4, 64, seed=sum(new) + sum(cached)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 1000, 2 ** 31 - 1])
def test_windows(odla, kind, window):
    announce("paged attention %s window %d" % (kind, window))
    check(odla, Case(kind, [1, 50, 150, 1], [300, 0, 40, 2000], 1, 3, 64, page=20, window=window, seed=window % 1000))


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_of_odd_pages_beyond_a_wavefront(odla, kind):
    """More than a wavefront has lanes, some of them without new tokens."""
    announce("paged attention %s of 150 sequences" % kind)
    rng = np.random.default_rng(4)
    check(odla, Case(kind, rng.integers(0, 4, 150), rng.integers(0, 200, 150), 2, 2, 16, page=7, seed=9))


@pytest.mark.parametrize("kind", KINDS)
def test_long_sequences_are_cut(odla, kind):
    announce("paged attention %s over 20000 places" % kind)
    check(odla, Case(kind, [1, 2], [20000, 7000], 1, 4, 64, page=32, seed=3), repeats=2)


@pytest.mark.parametrize("kind", KINDS)
def test_equal_sequences_need_no_starts(odla, kind):
    announce("paged attention %s without starts" % kind)
    check(odla, Case(kind, [3, 3, 3, 3], [0, 100, 7, 64], starts=False, seed=1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,cached", [([1, 1], [70, 400]), ([40, 3], [0, 50])])
def test_keys_that_lie_in_the_cache_already(odla, kind, new, cached):
    announce("paged attention %s without new keys" % kind)
    check(odla, Case(kind, new, cached, fresh=False, seed=2))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [3, 40], [150, 1]])
def test_tokens_of_no_sequence_give_zeros(odla, kind, new):
    announce("paged attention %s with tokens behind the last sequence" % kind)
    c = Case(kind, new, [30, 5], tail=6, seed=2)
    y = check(odla, c)
    assert not np.any(R.values(y[sum(new):], kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("junk", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new,window", [([1, 1, 2], 0), ([30, 5, 1], 0), ([140, 1, 1], 60)])
def test_what_no_token_owns_has_no_influence(odla, kind, junk, new, window):
    announce("paged attention %s beside %s" % (kind, junk))
    check(odla, Case(kind, new, [40, 3, 0], 1, 4, 64, junk=junk, window=window, seed=5))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [12, 150])
@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_keys_and_values_reach_the_tokens_that_see_them_alone(odla, kind, n, window, bad):
    """An infinite or missing value (or key) of one token: tokens in front of it, and those whose window has left it behind,
    are as if it were not there."""
    announce("paged attention %s, %d tokens, window %d, one %s" % (kind, n, window, bad))
    for part in ("v", "k"):
        c = Case(kind, [n], [3], 1, 2, 64, window=window, seed=6)
        at = n // 2
        getattr(c, part)[at, 0, 7] = R.to_bits(np.full(1, bad), kind)[0]
        y, kc, vc = run(odla, c)
        with np.errstate(invalid="ignore"):
            want, bound, _, _ = c.want()
        have = R.values(y, kind)
        sees = np.zeros(n, bool)
        sees[at:at + window if window else n] = True
        assert np.all(np.abs(have[~sees] - want[~sees]) <= bound[~sees]), part
        if part == "v":
            assert not np.any(np.isfinite(have[sees][:, :, 7]))
            if np.isinf(bad):
                assert np.all(have[sees][:, :, 7] == np.inf)
            rest = [i for i in range(64) if i != 7]
            assert np.all(np.abs(have[sees][:, :, rest] - want[sees][:, :, rest]) <= bound[sees][:, :, rest])
        elif np.isnan(bad):
            assert np.all(np.isnan(have[sees]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 140, 1]])
def test_pages_that_do_not_exist_are_neither_written_nor_seen(odla, kind, new):
    announce("paged attention %s with pages out of range" % kind)
    c = Case(kind, new, [70, 40, 9], 1, 4, 64, seed=8)
    pages = c.kc.shape[0]
    c.table[0, 1] = pages
    c.table[0, 3] = -5
    c.table[1, 0] = 2 ** 31 - 1
    c.table[1, 4] = -2 ** 31
    c.table[2] = -1                       # nothing of the last sequence exists
    y = check(odla, c)
    assert not np.any(R.values(y[sum(new[:2]):], kind))


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_beyond_the_table(odla, kind):
    """Places that the page table does not reach are neither written nor seen, negative lengths are none."""
    announce("paged attention %s with lengths out of range" % kind)
    c = Case(kind, [2, 3, 1], [30, 0, 60], 1, 2, 32, seed=8)
    reach = c.table.shape[1] * 16
    c.table[:] = np.random.default_rng(1).permutation(c.kc.shape[0])[np.arange(c.table.size) % c.kc.shape[0]].reshape(c.table.shape)
    for i in range(3):                    # a page in one sequence each
        c.table[i] = np.where(np.arange(c.table.size).reshape(c.table.shape)[i] < c.kc.shape[0], c.table[i], -1)
    c.cached[:] = [reach - 1, -7, 2 ** 31 - 1]
    check(odla, c)


def test_starts_out_of_range_stay_inside(odla):
    """Starts are clamped to the tokens that there are; what decreasing ones give has no meaning, but every launch ends inside
    its operands."""
    announce("paged attention with starts out of range")
    c = Case("bf16", [4, 4], [20, 3], 1, 2, 32, seed=8)
    c.starts = np.array([-3, 4, 1000], np.int32)
    y = run(odla, c)[0]
    c.starts = np.array([0, 4, 8], np.int32)
    assert np.array_equal(y, run(odla, c)[0])
    for odd in ([5, 2, 7], [8, 8, 0], [2 ** 31 - 1, -2 ** 31, 4]):
        c.starts = np.array(odd, np.int32)
        run(odla, c)


def test_scales(odla):
    announce("paged attention with other scales")
    for scale in (0.0, -0.3, 1.0, 30.0):
        check(odla, Case("fp32", [1, 5], [60, 3], d=16, scale=scale, seed=2))
        check(odla, Case("bf16", [1, 50], [60, 3], d=16, scale=scale, seed=2))


def test_captured_and_replayed(odla):
    """Graphs of several sets of buffers in turn, each with its own caches."""
    announce("paged attention captured for three sets of caches")
    cases = [Case("bf16", [1, 1, 4], [100, 7, 30], seed=s) for s in range(3)]
    b = odla.HipBuilder()
    feeds = [c.feeds(odla) for c in cases]
    b.output(cases[0].record(odla, b), "y")
    s = b.session()
    for k in (0, 1, 0, 2, 1, 2, 0):
        f = dict(feeds[k], pt=cases[k].table)
        have = R.values(s.run(f)["y"], "bf16")
        want, bound, kc, vc = cases[k].want()
        assert np.all(np.abs(have - want) <= bound), k
        assert np.array_equal(R.values(f["kc"].get(), "bf16"), kc)
    s.close()
    b.destroy()
    for f in feeds:
        f["kc"].close()
        f["vc"].close()


def test_a_sequence_grows(odla):
    """A prompt, then token after token, each execution extending the cache of the last: as one attention over all of them."""
    announce("paged attention, a prompt and twelve tokens behind it")
    kind, n, more, h, g, d, page = "fp32", 21, 12, 2, 3, 32, 4
    whole = Case(kind, [n + more], [0], h, g, d, page, seed=7)
    want, bound, kc, vc = whole.want()
    kc0, vc0 = odla.DeviceArray(whole.kc), odla.DeviceArray(whole.vc)
    got = []
    for first, t in [(0, n)] + [(n + i, 1) for i in range(more)]:
        part = Case(kind, [t], [first], h, g, d, page, seed=1)
        part.q, part.k, part.v = (a[first:first + t] for a in (whole.q, whole.k, whole.v))
        part.kc, part.vc, part.table = whole.kc, whole.vc, whole.table
        b = odla.HipBuilder()
        b.output(part.record(odla, b), "y")
        s = b.session()
        got.append(s.run({"q": part.q, "k": part.k, "v": part.v, "kc": kc0, "vc": vc0, "pt": part.table, "n": part.cached, "s": part.starts})["y"])
        s.close()
        b.destroy()
    assert np.all(np.abs(np.concatenate(got) - want) <= bound)
    assert np.array_equal(kc0.get(), kc) and np.array_equal(vc0.get(), vc)
    kc0.close()
    vc0.close()


@pytest.mark.parametrize("mode", [{"fp16": True}, {"bf16": True}, {"bf16": "accuracy"}])
def test_precision_modes_leave_caches_as_they_are_declared(odla, mode):
    """FLOAT32 caches stay fp32 in the modes that store other values in 16 bits, and bf16 ones bf16."""
    announce("paged attention, FLOAT32 caches, %s" % mode)
    kind = "fp16" if "fp16" in mode else "bf16"
    c = Case("fp32", [1, 6], [50, 3], seed=3)
    for n in "qkv":
        setattr(c, n, R.values(R.to_bits(getattr(c, n), kind), kind).astype(np.float32))     # (values that the mode's type holds)
    check(odla, c, **mode)
    check(odla, Case("bf16", [1, 6], [50, 3], seed=3), **mode)


def test_two_attentions_share_a_cache(odla):
    """The second reads what the first has written."""
    announce("two attentions over one cache")
    c = Case("bf16", [2, 1], [20, 40], seed=3)
    b = odla.HipBuilder()
    y = c.record(odla, b)
    b.output(y, "y")
    q2 = R.to_bits(np.random.default_rng(8).standard_normal(c.q.shape), "bf16")
    h = lambda n: b.args[n][0]
    b.output(b.paged_attention(b.arg("q2", q2.shape, odla.BFLOAT16), None, None, h("kc"), h("vc"), h("pt"), h("n"), h("s"), c.scale, name="y2"), "y2")
    feeds = dict(c.feeds(odla), q2=q2)
    s = b.session()
    got = s.run(feeds)
    s.close()
    b.destroy()
    want, bound, _, _ = c.want()
    assert np.all(np.abs(R.values(got["y"], "bf16") - want) <= bound)
    c.q = q2
    want, bound, _, _ = c.want()
    assert np.all(np.abs(R.values(got["y2"], "bf16") - want) <= bound)
    feeds["kc"].close()
    feeds["vc"].close()


def test_caches_that_cannot_be_extended_are_refused(odla):
    """Host memory, an address that is not aligned, and one buffer for both."""
    announce("caches that are refused")
    c = Case("bf16", [1], [5], seed=3)
    b = odla.HipBuilder()
    b.L.odla_SetLogLevel(0)
    b.output(c.record(odla, b), "y")
    s = b.session()
    feeds = c.feeds(odla)
    good = dict(feeds)
    import ctypes
    off = odla.DeviceArray(np.zeros(c.kc.nbytes + 64, np.uint8))
    try:
        for bad in (c.kc, feeds["vc"]):
            with pytest.raises(odla.OdlaError):
                s.run(dict(feeds, kc=bad))
        s.run(good)
        assert b.L.odla_BindToArgument(b.args["kc"][0], ctypes.c_void_p(off.ptr.value + 8), s.ctx) == 0
        with pytest.raises(odla.OdlaError):
            s.execute()
        s.run(good)
    finally:
        b.L.odla_SetLogLevel(2)
        s.close()
        b.destroy()
        off.close()
        feeds["kc"].close()
        feeds["vc"].close()


def test_static_execution(odla):
    """odla_hip_ExecuteComputationStatic extends the caches in place too."""
    announce("paged attention through the static entry point")
    c = Case("bf16", [1, 3], [50, 3], seed=3)
    b = odla.HipBuilder()
    b.output(c.record(odla, b), "y")
    s = b.session()
    feeds = c.feeds(odla)
    y = s.run(feeds)["y"]
    out = np.zeros_like(y)
    assert b.L.odla_BindToOutput(b.outs["y"][0], out.ctypes.data, s.ctx) == 0
    held = [np.ascontiguousarray(a) for a in (c.q, c.k, c.v, c.table, c.cached, c.starts)]
    for n, a in zip(("q", "k", "v", "pt", "n", "s"), held):
        assert b.L.odla_BindToArgument(b.args[n][0], a.ctypes.data, s.ctx) == 0
    assert s.execute_static() == 0
    assert np.array_equal(out, y)
    s.close()
    b.destroy()
    feeds["kc"].close()
    feeds["vc"].close()


@pytest.mark.parametrize("batch", [1, 3, 8])
def test_dynamic_batch(odla, batch):
    announce("paged attention at batch %d of up to 8" % batch)
    whole = Case("bf16", [1] * 8, [5, 60, 0, 33, 200, 1, 16, 15], starts=False, seed=3)
    b = odla.HipBuilder(max_batch=8)
    kind = odla.BFLOAT16
    row = lambda n, a, t=kind: b.arg(n, (-1,) + a.shape[1:], t)
    b.output(b.paged_attention(row("q", whole.q), row("k", whole.k), row("v", whole.v), b.arg("kc", whole.kc.shape, kind), b.arg("vc", whole.vc.shape, kind),
                               row("pt", whole.table, np.int32), row("n", whole.cached, np.int32), scale=whole.scale), "y")
    s = b.session()
    s.set_batch(batch)
    feeds = whole.feeds(odla)
    for n in ("q", "k", "v", "pt", "n"):
        feeds[n] = feeds[n][:batch]
    got = R.values(s.run(feeds)["y"], "bf16")
    want, bound, _, _ = whole.want()
    assert np.all(np.abs(got - want[:batch]) <= bound[:batch])
    s.close()
    b.destroy()
    feeds["kc"].close()
    feeds["vc"].close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [24, 80, 96, 192, 248])
@pytest.mark.parametrize("junk", [np.nan, np.inf])
def test_head_sizes_between_the_tiles(odla, kind, d, junk):
    """Few and many rows; the places that no sequence owns, some of them in the last pages read, hold no number."""
    announce("paged attention %s heads of %d among %s" % (kind, d, junk))
    check(odla, Case(kind, [1, 50, 3], [70, 21, 0], 2, 3, d, page=24, seed=d, junk=junk))
    check(odla, Case(kind, [2, 1], [300, 90], 1, 8, d, page=8, seed=d + 1, window=77, junk=junk))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 127, 128, 129])
@pytest.mark.parametrize("page", [8, 12, 36, 128])
def test_around_the_tiles_of_rows(odla, kind, rows, page):
    """Enough keys for several stretches of both ways of cutting."""
    announce("paged attention %s %d rows, pages of %d" % (kind, rows, page))
    check(odla, Case(kind, [rows, 1], [701, 1030], 1, 1, 64, page=page, seed=rows))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 150])
def test_a_long_chunk_behind_a_long_prompt(odla, kind, window):
    announce("paged attention %s a chunk of 410 behind 1500, window %d" % (kind, window))
    check(odla, Case(kind, [410], [1500], 1, 4, 128, page=20, seed=window, window=window))


@pytest.mark.parametrize("kind,d", [("fp16", 96), ("bf16", 128), ("fp32", 64)])
def test_every_execution_gives_the_same_bits(odla, kind, d):
    """A chunk whose tiles are many, cut, and as long as the memory is far: what has not landed in LDS yet would show."""
    announce("paged attention %s, heads of %d, 40 executions" % (kind, d))
    c = Case(kind, [509] + [1] * 8, [2500] + [600] * 8, 4, 4, d, page=32, seed=d)
    b = odla.HipBuilder()
    b.output(c.record(odla, b), "y")
    s = b.session()
    feeds = c.feeds(odla)
    first = s.run(feeds)["y"]
    again = [np.array_equal(s.run(feeds)["y"], first) for _ in range(40)]
    s.close()
    b.destroy()
    feeds["kc"].close()
    feeds["vc"].close()
    assert all(again), again


@pytest.mark.parametrize("new", [[1, 1], [40, 1]])
def test_caches_of_more_than_4_gib(odla, new):
    """Pages on both sides of 2 and 4 GiB, read and written."""
    import ctypes
    announce("paged attention over caches of 5 GiB, %s new tokens" % new)
    c = Case("bf16", new, [130, 200], 8, 1, 128, page=64, seed=len(new) + new[0])
    L, small, pages = odla.load_library(), c.kc.shape[0], 41000
    each = c.kc[0].nbytes
    assert (pages - 1) * each > 2 ** 32
    where = np.array([7, pages - 1, 2 ** 31 // each, 2 ** 31 // each - 1, 2 ** 32 // each, 2 ** 32 // each - 1, pages - 9, 0, 20000, 40000, 3, 33000])[:small]
    assert len(set(where)) == small

    def large(pages_of):
        a = odla.DeviceArray.__new__(odla.DeviceArray)
        a.L, a.shape, a.dtype, a.nbytes, a.ptr = L, (pages,) + pages_of.shape[1:], pages_of.dtype, pages * each, ctypes.c_void_p()
        assert L.odla_AllocateDeviceMemory(ctypes.byref(a.ptr), a.nbytes) == 0
        for i, at in enumerate(where):
            assert L.odla_CopyMemory(ctypes.c_void_p(a.ptr.value + int(at) * each), pages_of[i].ctypes.data_as(ctypes.c_void_p), each, odla.ODLA_MEMCPY_H2D) == 0
        return a

    def pages_back(a):
        got = np.empty_like(c.kc)
        for i, at in enumerate(where):
            assert L.odla_CopyMemory(got[i].ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(a.ptr.value + int(at) * each), each, odla.ODLA_MEMCPY_D2H) == 0
        return got

    want, bound, _, _ = c.want()
    kc_want, vc_want = c.written()
    kc, vc = large(c.kc), large(c.vc)
    b = odla.HipBuilder()
    kind = odla.BFLOAT16
    try:
        arg = lambda n, a: b.arg(n, a.shape, kind)
        b.output(b.paged_attention(arg("q", c.q), arg("k", c.k), arg("v", c.v), arg("kc", kc), arg("vc", vc), b.arg("pt", c.table.shape, np.int32),
                                   b.arg("n", (2,), np.int32), b.arg("s", (3,), np.int32), c.scale, 0, "y"), "y")
        s = b.session()
        y = s.run({"q": c.q, "k": c.k, "v": c.v, "kc": kc, "vc": vc, "pt": np.where(c.table < 0, -1, where[c.table]).astype(np.int32), "n": c.cached, "s": c.starts})["y"]
        s.close()
        assert np.array_equal(pages_back(kc), kc_want) and np.array_equal(pages_back(vc), vc_want)
    finally:
        b.destroy()
        kc.close()
        vc.close()
    assert np.all(np.abs(R.values(y, "bf16") - want) <= bound)


@pytest.mark.parametrize("kind,group", [("bf16", 2), ("fp32", 1)])
@pytest.mark.parametrize("b", [63, 64, 65, 255, 256, 257, 1000, 4200])
def test_many_sequences(odla, kind, group, b):
    """More sequences than lanes: single tokens, none, chunks of both ways of cutting, some cut into stretches; then one token each."""
    announce("paged attention %s of %d sequences" % (kind, b))
    rng = np.random.default_rng(b)
    new, cached = np.ones(b, int), rng.integers(0, 30, b)
    new[rng.random(b) < 0.2] = 0
    new[rng.integers(0, b, 6)] = 25
    cached[rng.integers(0, b, 4)] = 1200
    new[0], new[-1], cached[-1] = 0, 3, 900
    check(odla, Case(kind, new.tolist(), cached.tolist(), 1, group, 16, page=16, seed=b, tail=2))
    check(odla, Case(kind, [1] * b, cached.tolist(), 1, group, 16, page=16, seed=b + 1, starts=False))


class Logged:
    """The library's messages."""

    def __init__(self, odla):
        from test_gpu_device_args import capture_log
        self.L, self.seen = odla.load_library(), []
        self.keep = capture_log(self.L, self.seen)

    def count(self, part):
        return sum(part in m for m in self.seen)

    def close(self):
        self.L.odla_SetLogLevel(2)
        self.L.odla_SetLogger(None)


def run_in_turn(odla, cases, order, new_queries=False):
    """One context over the caches of `cases` in turn, queries in device memory: a buffer a case, or one an execution."""
    b = odla.HipBuilder()
    feeds = [dict(c.feeds(odla), q=odla.DeviceArray(c.q)) for c in cases]
    b.output(cases[0].record(odla, b), "y")
    s = b.session()
    log, wants, extra = Logged(odla), [c.want() for c in cases], []
    try:
        for k, i in enumerate(order):
            f = dict(feeds[i], pt=cases[i].table)
            if new_queries:
                extra.append(odla.DeviceArray(cases[i].q))
                f["q"] = extra[-1]
            have = R.values(s.run(f)["y"], cases[i].kind)
            want, bound, _, _ = wants[i]
            assert np.all(np.abs(have - want) <= bound), (k, i)
        for c, f in [(cases[i], feeds[i]) for i in sorted(set(order))]:
            kc, vc = c.written()
            assert np.array_equal(f["kc"].get(), kc) and np.array_equal(f["vc"].get(), vc)
        return log
    finally:
        log.close()
        s.close()
        b.destroy()
        for a in [a for f in feeds for a in f.values() if isinstance(a, odla.DeviceArray)] + extra:
            a.close()


def test_more_caches_in_turn_than_a_context_keeps_graphs(odla, monkeypatch):
    """A layer's computation over the caches of sixteen layers: after eight captures in a row executions run uncaptured, and
    operands are read in place still; with the same caches twice in a row captures are worth their while again."""
    announce("paged attention over sixteen pairs of caches in turn")
    monkeypatch.setenv("ODLA_HIP_GRAPH_MIN_STEPS", "1")
    cases = [Case("bf16", [1, 1, 4], [100, 7, 30], seed=s) for s in range(16)]
    log = run_in_turn(odla, cases, list(range(16)) * 3)
    assert log.count("copied from now on") == 0 and log.count("run uncaptured from now on") == 1
    assert log.count("launches captured") == 8
    assert log.count("argument 'q' is read in place") == 48
    log = run_in_turn(odla, cases, list(range(16)) * 2 + [3] * 6 + [5, 3, 3, 5])
    assert log.count("copied from now on") == 0 and 9 <= log.count("launches captured") <= 11


def test_new_operands_over_one_pair_of_caches_are_copied(odla, monkeypatch):
    """Other queries with every execution, the caches where they were: one graph over copies, as without caches."""
    announce("paged attention, new queries with every execution")
    monkeypatch.setenv("ODLA_HIP_GRAPH_MIN_STEPS", "1")
    cases = [Case("bf16", [1, 1, 4], [100, 7, 30], seed=s) for s in range(2)]
    for order, graphs in ([0] * 14, 1), ([0, 1] * 9, 2):
        log = run_in_turn(odla, cases, order, new_queries=True)
        assert log.count("copied from now on") == 1 and log.count("uncaptured") == 0
        assert log.count("launches captured") == 8 + graphs


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,cached,window", [([1], [100], 0), ([3, 1], [5000, 70], 0), ([1], [40000], 0), ([40], [600], 0), ([150], [200], 0), ([150], [3000], 0),
                                               ([150], [200], 120), ([5], [300], 90)])
def test_infinite_values_count_however_small_their_weights(odla, kind, new, cached, window):
    """With a scale of 30 nearly all weights are too small for 32 bits.  A value that is no number reaches every row that sees it all the same:
    in tiles that all rows see and in those with a mask, in front of the maximum and behind it, in every part of a row that is cut."""
    announce("paged attention %s, %s behind %s, window %d, infinite values of no weight" % (kind, new, cached, window))
    rng = np.random.default_rng(cached[0] + new[0])
    for bad in (np.inf, -np.inf, np.nan, "both"):
        c = Case(kind, new, cached, 1, 2, 64, scale=30.0, window=window, seed=7)
        n, total = new[0], new[0] + cached[0]
        odd = {}      # column -> {place: value}
        for column in (0, 7, 34, 63):
            for value in (np.inf, -np.inf) if bad == "both" else (bad,):
                place = int(rng.integers(max(0, cached[0] - 80) if window else 0, total))
                odd.setdefault(column, {})[place] = value
                bits = R.to_bits(np.full(1, value), kind)[0]
                if place < cached[0]:
                    c.vc[c.table[0, place // 16], place % 16, 0, column] = bits
                else:
                    c.v[place - cached[0], 0, column] = bits
        y, _, _ = run(odla, c)
        with np.errstate(invalid="ignore", over="ignore"):
            want, bound, _, _ = c.want()
        have = R.values(y, kind)
        for column, values in odd.items():
            for i in range(n):
                p = cached[0] + i
                seen = [v for at, v in values.items() if at <= p and (window == 0 or at > p - window)]
                if not seen:
                    continue
                with np.errstate(invalid="ignore"):
                    total_of = np.sum(seen)
                for h in range(2):
                    got = have[i, h, column]
                    assert got == total_of or (np.isnan(got) and np.isnan(total_of)), (bad, column, i, h, got, total_of)
                    want[i, h, column], bound[i, h, column], have[i, h, column] = 0, 0, 0
        assert np.all(np.abs(have - want) <= bound), bad


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("seqs,new,heads,n", [(1, 8192, 8, 57344), (64, 1, 16, 16384)])
def test_many_keys_of_little_weight_add_up(odla, kind, seqs, new, heads, n):
    """A first key of weight 1 whose value is 0, and tens of thousands of weight exp(-17.75) = 2^-25.6 and value 1 behind it in the same piece: they are
    a thousandth, which is all of the result.  An fp16 weight is off by 2^-25 of 2^7 at most there, all of them by their number times 2^-32."""
    announce("paged attention %s, %d x %d tokens, %d keys of little weight" % (kind, seqs, new, n))
    d, page = 8, 64
    b = odla.HipBuilder()
    dtype = np_kind(odla, kind)
    pages = -(-(n + new) // page)
    k, v = np.zeros((pages, page, heads, d)), np.ones((pages, page, heads, d))
    k[..., 0] = -17.75
    k[0, 0], v[0, 0] = 0, 0
    q = np.zeros((seqs * new, heads, d))
    q[..., 0] = 1
    feeds = {"q": R.to_bits(q, kind), "kc": odla.DeviceArray(R.to_bits(k, kind)), "vc": odla.DeviceArray(R.to_bits(v, kind)),
             "pt": np.tile(np.arange(pages, dtype=np.int32), (seqs, 1)), "n": np.full(seqs, n, np.int32)}      # (the new tokens' keys are there already)
    h = {x: b.arg(x, feeds[x].shape, np.int32 if x in ("pt", "n") else dtype) for x in feeds}
    b.output(b.paged_attention(h["q"], None, None, h["kc"], h["vc"], h["pt"], h["n"], scale=1.0, name="y"), "y")
    s = b.session()
    have = R.values(s.run(feeds)["y"], kind).reshape(seqs, new, heads * d)
    s.close()
    b.destroy()
    feeds["kc"].close()
    feeds["vc"].close()
    keys = n + np.arange(new)[None, :, None]
    total = 1 + keys * np.exp(-17.75)
    want = keys * np.exp(-17.75) / total
    # (exponentials of a distance of 17.75, and sums of as many terms in fp32, each off by 2^-24 of what is there; the weights' and the result's type)
    bound = (R.EPS[kind] / 2 * (1 if kind == "fp32" else 2) + (4 * 17.75 + 8 + 2 * keys / 32) * L.ULP) * want + R.LEAST[kind] + (keys * 2.0 ** -32 / total if kind == "fp16" else 0)
    assert np.all(np.abs(have - want) <= bound), np.max(np.abs(have - want) / bound)
