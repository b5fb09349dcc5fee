"""CPU: what dn_host_register answers when hipHostRegister refuses.  A child process loads a stand-in for the four runtime calls in front of the library (its symbols
are found first), so that every refusal can be had without a device."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STAND_IN = """
static int next_, last_, registered_;
void answer(int e) { next_ = e; }
int registered(void) { return registered_; }
int last(void) { return last_; }
int hipHostRegister(void *p, unsigned long n, unsigned f) { (void)p; (void)n; (void)f; if (next_) last_ = next_; else registered_++; return next_; }
int hipHostUnregister(void *p) { (void)p; if (!registered_) { last_ = 713; return 713; } registered_--; return 0; }
int hipGetLastError(void) { int e = last_; last_ = 0; return e; }
"""
CHILD = """
import ctypes as C, sys
sys.path.insert(0, %r)
stand = C.CDLL(%r, C.RTLD_GLOBAL)
from dnascent_amd import hip
L = hip.lib()
buf = C.create_string_buffer(1 << 16)
p, n = C.addressof(buf), 1 << 16
OK, HIP, ARG = 0, -2, -3
def ask(e, p=p, n=n):
    stand.answer(e)
    rc = L.dn_host_register(p, n)
    assert stand.last() == 0, "an error is left for the next call"
    return rc
%s
print("fine")
"""
NO_DEVICE, OUT_OF_MEMORY, INVALID, NOT_SUPPORTED, ALREADY = 100, 2, 1, 801, 712


def run(tmp_path, body):
    so = tmp_path / "stand_in.so"
    (tmp_path / "stand_in.c").write_text(STAND_IN)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(so), str(tmp_path / "stand_in.c")])
    got = subprocess.run([sys.executable, "-c", CHILD % (ROOT, str(so), body)], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "fine", got.stderr


@pytest.mark.parametrize("e", [NO_DEVICE, OUT_OF_MEMORY, ALREADY])
def test_other_failures_are_errors(tmp_path, e):
    run(tmp_path, "assert ask(%d) == HIP and L.dn_host_unregister(p) == HIP" % e)


@pytest.mark.parametrize("e", [INVALID, NOT_SUPPORTED])
def test_refused_memory_stays_pageable(tmp_path, e):
    run(tmp_path, "assert ask(%d) == OK and ask(%d) == OK\n"
                  "assert [L.dn_host_unregister(p) for _ in range(3)] == [OK, OK, HIP] and stand.registered() == 0" % (e, e))


def test_a_range_that_is_not_there_is_an_error(tmp_path):
    run(tmp_path, "import mmap\n"
                  "m = mmap.mmap(-1, 8 * 4096)\n"
                  "c = (C.c_char * len(m)).from_buffer(m); at = C.addressof(c)\n"
                  "assert ask(%d, at, 8 * 4096) == OK and L.dn_host_unregister(at) == OK\n"
                  "del c; m.close()\n"
                  "assert ask(%d, at, 8 * 4096) == HIP and ask(%d, 4096, 4096) == HIP and ask(%d, p, 2**64 - 1 - p) == HIP and ask(%d, p, 2**64 - 1) == HIP\n"
                  "assert ask(0, 0, 5) == ARG and ask(0, p, 0) == ARG" % ((INVALID,) * 5))


def test_a_stale_refusal_does_not_keep_memory_locked(tmp_path):
    """refused, freed without dn_host_unregister, and the address registered for good later: dn_host_unregister means the registration"""
    run(tmp_path, "assert ask(%d) == OK and ask(%d) == OK and ask(0) == OK and stand.registered() == 1\n"
                  "assert L.dn_host_unregister(p) == OK and stand.registered() == 0 and L.dn_host_unregister(p) == HIP" % (INVALID, INVALID))
