"""CPU test of when the Python entry of the operators is built again (momij_b200/build.py)."""
from __future__ import annotations

import os

from momij_b200 import build


def test_binding_is_rebuilt_for_another_torch(tmp_path):
    src, out, stamp = (str(tmp_path / n) for n in ("bind.cpp", "ops.so", "bind.stamp"))
    for i, f in enumerate((src, out)):
        open(f, "w").close()
        os.utime(f, (1000 + i, 1000 + i))
    assert not build._bind_is_current(out, [src], stamp, "torch A")  # built by nobody knows what
    with open(stamp, "w") as f:
        f.write("torch A")
    assert build._bind_is_current(out, [src], stamp, "torch A")
    assert not build._bind_is_current(out, [src], stamp, "torch B")
    os.utime(src, (2000, 2000))
    assert not build._bind_is_current(out, [src], stamp, "torch A")
    os.remove(out)
    assert not build._bind_is_current(out, [src], stamp, "torch A")
