"""Properties of the compiled gfx950 code of the kernels over 8-bit blocks, experts' weights and logits that their
correctness relies on: buffer loads whose range check needs nothing but a lane's offset, and nothing on its way
into LDS where wavefronts meet."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import __graft_entry__ as entry

HIPCC = "/opt/rocm/bin/hipcc"
KERNELS = os.path.join(entry.ROOT, "heterogeneity-aware-lowering-and-optimization_amd", "csrc", "kernels")
FLAGS = ["--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-O3", "-std=c++17",
         "-fPIC", "-ffp-contract=off", "--cuda-device-only", "-S"]
FILES = ("block_fp8", "experts", "sample")


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    """Instructions and labels of every kernel of the three files."""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("block_asm")

    def compile_one(f):
        out = os.path.join(d, f + ".s")
        r = subprocess.run([HIPCC] + FLAGS + [os.path.join(KERNELS, f + ".hip"), "-o", out], capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-2000:]
        return open(out).read()

    found = {}
    with ThreadPoolExecutor(len(FILES)) as pool:
        for asm in pool.map(compile_one, FILES):
            for name in re.findall(r"^(_ZN4ohip\w+):", asm, re.M):
                a = asm.index("\n" + name + ":")
                body = [l.split(";")[0].strip() for l in asm[a:asm.index(".Lfunc_end", a)].split("\n")[2:]]
                found[name] = [l for l in body if l and (not l.startswith(".") or l.startswith(".LBB"))]
    assert len(found) > 80
    return found


def test_ranges_are_checked_against_lane_offsets_alone(bodies):
    """A scalar offset beyond a buffer's size has no defined meaning in its check: no load has one."""
    seen = 0
    for name, body in bodies.items():
        for l in body:
            if l.startswith("buffer_load"):
                seen += 1
                assert re.search(r", s\[\d+:\d+\], 0 offen\b", l), (name, l)
    assert seen > 500


def is_lds_write(op, l):
    return op.startswith("ds_") and ("write" in op or "add" in op or "append" in op)


def is_load_into_lds(op, l):
    return op.startswith(("buffer_load", "global_load")) and bool(re.search(r"\blds\b|_lds_", l))


def unsettled_barrier(body, starts=is_lds_write, counter="lgkmcnt"):
    """The first s_barrier that some path reaches with what `starts` names not waited for, or None.  (Only a wait for 0
    settles the last of them.)"""
    labels = {l[:-1]: i for i, l in enumerate(body) if l.endswith(":")}
    wait = re.compile(r"s_waitcnt\b.*%s\(0\)" % counter)
    dirty_at = [None] * len(body)      # whether a write may be under way in front of instruction i: unknown, False or True
    todo = [(0, False)]
    while todo:
        i, dirty = todo.pop()
        while i < len(body):
            if dirty_at[i] is not None and (dirty_at[i] or not dirty):
                break
            dirty_at[i] = dirty
            l = body[i]
            op = l.split()[0]
            if wait.match(l) or l.strip() == "s_waitcnt 0":
                dirty = False
            elif starts(op, l):
                dirty = True
            elif op == "s_barrier" and dirty:
                return i
            if op == "s_endpgm":
                break
            if op.startswith("s_cbranch") or op == "s_branch":
                target = labels[l.split()[1]]
                todo.append((target, dirty))
                if op == "s_branch":
                    break
            i += 1
    return None


def test_the_walk_over_barriers():
    assert unsettled_barrier(["ds_write_b32 v0, v1", "s_barrier", "s_endpgm"]) == 1
    assert unsettled_barrier(["ds_write_b32 v0, v1", "s_waitcnt vmcnt(0) lgkmcnt(0)", "s_barrier", "s_endpgm"]) is None
    loop = [".LBB0_1:", "s_waitcnt vmcnt(0)", "s_barrier", "ds_write_b32 v0, v1", "s_cbranch_scc0 .LBB0_1", "s_endpgm"]
    assert unsettled_barrier(loop) == 2                      # (the write of the turn before)
    assert unsettled_barrier(loop[:4] + ["s_waitcnt lgkmcnt(0)"] + loop[4:]) is None
    direct = ["buffer_load_dwordx4 v1, s[4:7], 0 offen lds", "s_waitcnt lgkmcnt(0)", "s_barrier", "s_endpgm"]
    assert unsettled_barrier(direct, is_load_into_lds, "vmcnt") == 2 and unsettled_barrier(direct) is None


def test_lds_writes_are_settled_in_front_of_every_barrier(bodies):
    barriers = 0
    for name, body in bodies.items():
        barriers += sum(l == "s_barrier" for l in body)
        at = unsettled_barrier(body)
        assert at is None, (name, body[max(0, at - 8):at + 1])
    assert barriers > 300


def test_loads_into_lds_are_settled_in_front_of_every_barrier(bodies):
    loads = 0
    for name, body in bodies.items():
        loads += sum(is_load_into_lds(l.split()[0], l) for l in body)
        at = unsettled_barrier(body, is_load_into_lds, "vmcnt")
        assert at is None, (name, body[max(0, at - 8):at + 1])
    assert loads >= 4 * 8
