"""Additions to the sampling's bins: what may lie behind the last bin is added by one function, which looks."""
import os
import re

import __graft_entry__ as entry


def test_bins_of_logits_are_checked():
    src = open(os.path.join(entry.PKG_DIR, "csrc", "kernels", "sample.hip")).read()
    body = re.search(r"void add_to_bin\(N\* bins, const int b, const N n\) \{\n(.*?)\n\}", src, re.S).group(1)
    assert re.search(r"if \(b < kBins\) atomicAdd\(&bins\[b\], n\);", body)
    direct = re.findall(r"atomicAdd\(&s\.(?:sum|count)\[(.*?)\], ", src)
    # a digit of a key (b = mask - digit), and parts of a row's indexes
    assert sorted(set(direct)) == ["b", "i / part", "kept_i[j] / part"], direct
    assert len(re.findall(r"atomicAdd\(&s\.(?:sum|count)\[b\]", src)) == 2 and src.count("const unsigned b = mask - ((k >> shift) & mask);") == 1
