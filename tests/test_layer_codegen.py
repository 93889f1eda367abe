"""The compiled gfx950 code of the kernels of a layer's operators: nothing is on its way into LDS where wavefronts meet."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_block_codegen import FLAGS, HIPCC, KERNELS, is_load_into_lds, unsettled_barrier

FILES = ("paged_attention", "log_probs", "rms_norm")


def kernels_of(asm):
    found = {}
    for name in re.findall(r"^(_ZN4ohip\w+):", asm, re.M):
        a = asm.index("\n" + name + ":")
        body = [l.split(";")[0].strip() for l in asm[a:asm.index(".Lfunc_end", a)].split("\n")[2:]]
        found[name] = [l for l in body if l and (not l.startswith(".") or l.startswith(".LBB"))]
    return found


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("layer_asm")

    def compile_one(f):
        out = os.path.join(d, f + ".s")
        r = subprocess.run([HIPCC] + FLAGS + [os.path.join(KERNELS, f + ".hip"), "-o", out], capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-2000:]
        return kernels_of(open(out).read())

    with ThreadPoolExecutor(len(FILES)) as pool:
        return {n: b for found in pool.map(compile_one, FILES) for n, b in found.items()}


def test_lds_is_settled_in_front_of_every_barrier(bodies):
    """Writes to LDS by their counter, loads into it by theirs: a barrier itself waits for neither."""
    loads = 0
    for name, body in bodies.items():
        loads += sum(is_load_into_lds(l.split()[0], l) for l in body)
        for at in (unsettled_barrier(body), unsettled_barrier(body, is_load_into_lds, "vmcnt")):
            assert at is None, (name, body[max(0, at - 8):at + 1])
    assert loads >= 8 * 20
