"""CPU test of a rule that the kernels' overlap rests on: a kernel that may start while
the one before it in the stream still runs waits for that on every path, since the
kernel after it waits for it alone."""
from __future__ import annotations

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "momij_b200", "csrc")


def kernels():
    """(file, name, body) of every __global__ function."""
    for f in sorted(os.listdir(CSRC)):
        if not f.endswith((".cu", ".cuh")):
            continue
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, f)).read())
        for m in re.finditer(r"__global__[^{;]*?(\w+)\s*\(([^()]*)\)\s*\{", text):
            depth, i = 1, m.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[i], 0)
                i += 1
            yield f, m.group(1), text[m.end():i]


def test_kernels_wait_for_the_one_before_on_every_path():
    seen = 0
    for f, name, body in kernels():
        wait = body.find("pdl_wait()")
        if wait < 0:
            continue
        seen += 1
        assert "return" not in body[:wait], f"{f}: {name} may end before its wait"
    assert seen >= 20


def test_a_kernel_without_the_wait_is_not_launched_to_overlap():
    waiting = {name for _, name, body in kernels() if "pdl_wait()" in body}
    for f in os.listdir(CSRC):
        text = open(os.path.join(CSRC, f)).read()
        for name in re.findall(r"\blaunch\(\s*(\w+_kernel)\b", text) + re.findall(r"host_launch\(\s*(\w+_kernel)\b", text):
            assert name in waiting, f"{f}: {name}"
