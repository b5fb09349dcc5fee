"""CPU: no packed fp32 arithmetic in the kernels -- some of its forms have given wrong results on this hardware now and then, which no test of results reliably shows."""
import glob
import os
import re

from dnascent_amd import build


def test_every_kernel_is_compiled_without_packed_fp32(monkeypatch):
    commands = []
    monkeypatch.setattr(build, "_run", commands.append)
    build.build_hip(force=True)
    compiled = [c for c in commands if "-c" in c]
    assert sorted(os.path.basename(c[c.index("-c") + 1]) for c in compiled) == sorted(build.HIP_SOURCES)
    for c in compiled:
        at = c.index("-packed-fp32-ops")
        assert c[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]


def test_no_kernel_writes_them_by_hand():
    files = [f for p in ("*.hip", "*.h") for f in glob.glob(os.path.join(build.CSRC, p))]
    assert len(files) >= 15
    for f in files:
        assert not re.search(r"v_pk_(fma|mul|add|mov)_(f32|b32)", open(f).read()), f
