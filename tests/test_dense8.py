"""CPU: what the 8-bit dense layers refuse.  The C entries' checks run through the workspace queries, which look at the description only; the torch
side's through tensors that never reach a device.  Nothing is launched."""
import ctypes as C
import os
import struct
import subprocess
from types import SimpleNamespace

import pytest
import torch

from dnascent_amd import dense8, hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                                                # an aligned address that nothing dereferences


def _linear(**kw):
    d = dict(m=5, n=7, k=33, x=P, ldx=33, sx=None, w=P, ldw=48, sw=P, bias=None, residual=None, ldr=0, y=P, ldy=7, mask=None, ldmask=0, q=None, ldq=0,
             s=None, x_type=0, y_type=0, relu=0, reserved=0)
    d.update(kw)
    return hip.i8_desc(hip.I8_LINEAR_FIELDS, **d)


def _grad(**kw):
    d = dict(m=5, n=7, k=33, dy=P, ldy=7, mask=None, ldmask=0, q=P, ldq=48, s=P, w=P, ldw=48, sw=P, dx=P, ldx=33, dw=P, lddw=33, db=P, dy_type=0, dw_type=0)
    d.update(kw)
    return hip.i8_desc(hip.I8_GRAD_FIELDS, **d)


def _ask(entry, d):
    need = C.c_uint64(0)
    return getattr(hip.lib(), entry + "_workspace")(None, d, C.byref(need)), need.value


@pytest.mark.parametrize("kw", [
    dict(), dict(m=0, x=None, y=None), dict(m=1, ldx=0), dict(ldx=0), dict(bias=P), dict(residual=P, ldr=7), dict(relu=1, mask=P, ldmask=1),
    dict(q=P, ldq=33, s=P), dict(x_type=3, sx=P), dict(x_type=1, y_type=2), dict(n=131071, ldy=131071), dict(k=131071, ldx=131071, ldw=131071),
    dict(m=2147483135), dict(ldx=1 << 21)])
def test_linear_takes(kw):
    assert _ask("dn_i8_linear", _linear(**kw))[0] == 0


@pytest.mark.parametrize("kw", [
    dict(m=-1), dict(m=2147483136), dict(n=0), dict(k=0), dict(n=131072, ldy=131072), dict(k=131072, ldx=131072, ldw=131072),     # sizes
    dict(x_type=4), dict(x_type=-1), dict(y_type=3), dict(relu=2), dict(reserved=1),                                               # types and flags
    dict(x=None), dict(w=None), dict(sw=None), dict(y=None), dict(x=P + 2), dict(y=P + 1), dict(sw=P + 2), dict(bias=P + 1),       # missing, misaligned
    dict(x_type=1, x=P + 1), dict(ldx=32), dict(ldx=-1), dict(ldw=32), dict(ldy=6), dict(ldy=0), dict(residual=P, ldr=3),          # pitches
    dict(m=1, ldy=6), dict(ldx=1 << 31), dict(ldx=(1 << 21) + 1),
    dict(x_type=3), dict(sx=P), dict(mask=P, ldmask=1), dict(relu=1, mask=P, ldmask=0), dict(q=P, ldq=33), dict(s=P), dict(q=P, ldq=32, s=P),
    dict(x_type=3, sx=P, q=P, ldq=33, s=P)])
def test_linear_refuses(kw):
    assert _ask("dn_i8_linear", _linear(**kw))[0] == -3


@pytest.mark.parametrize("kw", [
    dict(), dict(m=0, dy=None, q=None, s=None, dx=None), dict(dx=None), dict(dw=None, db=None), dict(dw=None), dict(db=None), dict(mask=P, ldmask=1),
    dict(dy_type=2, dw_type=0), dict(ldq=0), dict(ldy=0), dict(dx=None, w=None, sw=None), dict(dw=None, q=None, s=None)])
def test_grad_takes(kw):
    assert _ask("dn_i8_linear_grad", _grad(**kw))[0] == 0


@pytest.mark.parametrize("kw", [
    dict(m=-1), dict(n=0), dict(k=0), dict(k=131072, ldq=131072, ldw=131072, ldx=131072, lddw=131072), dict(dy_type=3), dict(dw_type=3), dict(dy=None),
    dict(dy=P + 2), dict(q=None), dict(s=None), dict(w=None), dict(sw=None), dict(dx=P + 2), dict(dw=P + 2), dict(db=P + 2), dict(ldx=32), dict(lddw=32),
    dict(ldq=32), dict(ldw=32), dict(ldy=6), dict(n=9, ldy=9, mask=P, ldmask=1), dict(dx=None, dw=None, db=None)])
def test_grad_refuses(kw):
    assert _ask("dn_i8_linear_grad", _grad(**kw))[0] == -3


@pytest.mark.parametrize("kw,rows", [(dict(ldw=297), 0), (dict(w=P + 1), 0), (dict(x=P + 8), 1), (dict(ldx=297), 1)])
def test_workspace_follows_addresses_and_pitches(kw, rows):
    """rows that do not lie at multiples of 16 bytes are copied to where they do (rows of more than 256 codes; narrower ones are read
    as they lie): 304 bytes for 297 codes, w's 300 rows or x's 200"""
    wide = dict(m=200, n=300, k=297, x=P, ldx=304, x_type=3, sx=P, ldw=304, ldy=300)
    rc, base = _ask("dn_i8_linear", _linear(**wide))
    wide.update(kw)
    rc2, need = _ask("dn_i8_linear", _linear(**wide))
    assert rc == rc2 == 0 and need - base == -(-(200 if rows else 300) * 304 // 256) * 256


def test_null_arguments():
    L = hip.lib()
    n = C.c_uint64(0)
    assert L.dn_i8_linear_workspace(None, None, C.byref(n)) == -3 and L.dn_i8_linear_workspace(None, _linear(), None) == -3
    assert L.dn_i8_linear(None, _linear(), None, 0, None) == -3 and L.dn_i8_linear_grad(None, _grad(), None, 0, None) == -3
    assert L.dn_i8_rows(None, 1, 1, P, 1, 0, P, 16, P, None) == -3 and L.dn_i8_restore(None, 1, 1, P, 16, P, P, 1, 0, None) == -3


def test_description_layouts_match_the_header(tmp_path):
    src = tmp_path / "layout.c"
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dnascent_hip.h"', 'int main(void) {']
    want = []
    for name, fields in (("dn_i8_linear_desc", hip.I8_LINEAR_FIELDS), ("dn_i8_grad_desc", hip.I8_GRAD_FIELDS)):
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f, _ in fields]
        code = "".join(f for _, f in fields)
        want += [struct.calcsize("@" + code)] + [struct.calcsize("@" + code[:i + 1]) - struct.calcsize("@" + code[i]) for i in range(len(code))]
    src.write_text("\n".join(lines + ['return 0; }']))
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    assert [int(v) for v in subprocess.check_output([str(exe)]).decode().split()] == want
    assert (hip.I8_LINEAR.size, hip.I8_GRAD.size) == (want[0], want[len(hip.I8_LINEAR_FIELDS) + 1])


def test_how_rows_lie():
    t = torch.zeros(6, 4, 10)
    assert dense8._rows("t", t) == (24, 10, 10)
    assert dense8._rows("t", t[:, :, :7]) == (24, 7, 10)
    assert dense8._rows("t", t[0, 0]) == (1, 10, 10)
    assert dense8._rows("t", t[:, 1]) == (6, 10, 40)
    assert dense8._rows("t", t[2:3, 1:2]) == (1, 10, 10)
    assert dense8._rows("t", torch.zeros(1, 10).expand(5, 10)) == (5, 10, 0)
    assert dense8._rows("t", torch.zeros(0, 10)) == (0, 10, 10)
    assert dense8._rows("t", torch.zeros(5, 8)[:, :1]) == (5, 1, 8)
    for bad in (t.transpose(1, 2), t[:, 1:3], t.transpose(0, 1), torch.zeros(3, 0), torch.zeros(()), torch.zeros(1).expand(5, 10),
                torch.zeros(40).as_strided((5, 10), (4, 1))):
        with pytest.raises(ValueError):
            dense8._rows("t", bad)
    q, pitch = dense8._empty_rows((3, 2, 33), "cpu")
    assert q.shape == (3, 2, 33) and dense8._rows("q", q) == (6, 33, 48) and pitch == 48
    q, pitch = dense8._empty_rows((5, 32), "cpu")
    assert q.shape == (5, 32) and dense8._rows("q", q) == (5, 32, 32) and pitch == 32


def test_tensors_of_another_device_are_refused():
    ctx = SimpleNamespace(device=0, h=None)
    x = torch.zeros(2, 8)
    q, s = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: dense8.rows(ctx, x), lambda: dense8.restore(ctx, q, s, torch.float32), lambda: dense8.linear(ctx, x, q, s),
                 lambda: dense8.linear_grad(ctx, x, q, s, q, s)):
        with pytest.raises(ValueError, match="context on device 0"):
            call()
    with pytest.raises(TypeError):
        dense8.rows(ctx, x.numpy())


def test_arguments_that_require_a_gradient_are_refused():
    """i8_linear, i8_linear_grad and i8_restore give tensors without a history; on tensors of no device, which the checks in front of the first call see"""
    ctx = SimpleNamespace(device=-1, h=None)
    x, q, s, b = torch.zeros(2, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3), torch.zeros(3)
    x8, sx, r = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2), torch.zeros(2, 3)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for name, call in [("x", lambda: dense8.linear(ctx, grad(x), q, s)), ("ws", lambda: dense8.linear(ctx, x, q, grad(s))), ("bias", lambda: dense8.linear(ctx, x, q, s, bias=grad(b))),
                       ("residual", lambda: dense8.linear(ctx, x, q, s, residual=grad(r))), ("sx", lambda: dense8.linear(ctx, x8, q, s, sx=grad(sx))),
                       ("s", lambda: dense8.restore(ctx, q, grad(s), torch.float32)), ("dy", lambda: dense8.linear_grad(ctx, grad(r), x8, sx, q, s))]:
        with pytest.raises(ValueError, match="^%s requires a gradient" % name):
            call()


def test_arguments_that_are_no_tensors_are_type_errors():
    ctx = SimpleNamespace(device=-1, h=None)
    x, q, s = torch.zeros(2, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: dense8.linear(ctx, x.numpy(), q, s), lambda: dense8.linear(ctx, x, q, s, bias=s.numpy()), lambda: dense8.linear(ctx, x, q, s, residual=[0.0]),
                 lambda: dense8.linear(ctx, torch.zeros(2, 8, dtype=torch.int8), q, s, sx=s.numpy()), lambda: dense8.linear_grad(ctx, x, torch.zeros(2, 8, dtype=torch.int8), 3.0, q, s)):
        with pytest.raises(TypeError):
            call()
