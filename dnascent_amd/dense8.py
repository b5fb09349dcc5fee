"""8-bit dense layers on torch tensors: the checks and allocations behind hip.Context.i8_*, and the layer that is trained with them.

A dense layer y = act(x W^T + b) over rows of x (positions of reads).  Its input and its weight are kept as rows of 8-bit integers with one fp32
scale each (include/dnascent_hip.h has the formulas); the same 8-bit rows are what the product multiplies and what its gradient needs, so a layer that
is being fitted keeps K + 4 bytes per row between forward and backward pass, and one bit per output if a ReLU follows, instead of numbers.
The reference has no counterpart: its network is a frozen SavedModel (tensor.cpp:12-106), trained outside it.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import hip

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}      # DN_T_*


class Saved(NamedTuple):
    """what a layer keeps for its gradient: q [..., K] int8, s [...] fp32, and mask [rows, (N + 7) // 8] uint8 (bit n % 8 of byte n // 8) or None"""
    q: torch.Tensor
    s: torch.Tensor
    mask: Optional[torch.Tensor]


def _check(ctx, name, t, dtypes, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: a torch tensor is expected, not %s" % (name, type(t).__name__))
    if t.device.type != "cuda" or t.device.index != ctx.device:
        raise ValueError("%s is on %s, the context on device %d" % (name, t.device, ctx.device))
    if t.dtype not in dtypes:
        raise TypeError("%s is %s" % (name, t.dtype))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has the shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _rows(name, t):
    """t [..., C] as (rows, C, pitch in elements): its elements stay where they are"""
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError("%s has the shape %s: rows of at least one element are expected" % (name, tuple(t.shape)))
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("%s: the elements of a row are not next to each other (call .contiguous())" % name)
    c = t.shape[-1]
    if t.dim() == 1:
        return 1, c, c
    m = t.numel() // c
    if m == 0:
        return 0, c, c
    lead = [(n, st) for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
    if not lead:
        return m, c, c
    for (_, outer), (n, inner) in zip(lead[:-1], lead[1:]):
        if outer != n * inner:
            raise ValueError("%s: its rows do not lie at one pitch (call .contiguous())" % name)
    pitch = lead[-1][1]
    if 0 < pitch < c:
        raise ValueError("%s: its rows overlap (call .contiguous())" % name)
    return m, c, pitch


def _vector(name, t, dtype=torch.float32):
    if t.numel() > 1 and not t.is_contiguous():
        raise ValueError("%s is not contiguous" % name)


def _stream(ctx):
    return torch.cuda.current_stream(ctx.device).cuda_stream


def _empty_rows(shape, device):
    """int8 [..., K] whose rows start at multiples of 16 bytes"""
    k = shape[-1]
    return torch.empty(*shape[:-1], (k + 15) // 16 * 16, dtype=torch.int8, device=device)[..., :k]


def _pitch(q):
    """row pitch of a tensor that _empty_rows made"""
    return (q.shape[-1] + 15) // 16 * 16


def _workspace(ctx, entry, desc):
    need = C.c_uint64(0)
    ctx._chk(getattr(hip.lib(), entry + "_workspace")(ctx.h, C.byref(desc), C.byref(need)), entry)
    return torch.empty(need.value, dtype=torch.uint8, device="cuda:%d" % ctx.device) if need.value else None, need.value


def _run(ctx, entry, desc):
    ws, need = _workspace(ctx, entry, desc)                # torch's allocator: the caller's stream, or the graph being captured, owns it
    ctx._chk(getattr(hip.lib(), entry)(ctx.h, C.byref(desc), ws.data_ptr() if ws is not None else None, need, _stream(ctx)), entry)


_NUMBERS = (torch.float32, torch.float16, torch.bfloat16)


def rows(ctx, x):
    _check(ctx, "x", x, _NUMBERS)
    m, k, ldx = _rows("x", x)
    q = _empty_rows(x.shape, x.device)
    s = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    ctx._chk(hip.lib().dn_i8_rows(ctx.h, m, k, x.data_ptr(), ldx, TYPES[x.dtype], q.data_ptr(), _pitch(q), s.data_ptr(), _stream(ctx)), "dn_i8_rows")
    return q, s


def restore(ctx, q, s, dtype):
    _check(ctx, "q", q, (torch.int8,))
    _check(ctx, "s", s, (torch.float32,), q.shape[:-1])
    _vector("s", s)
    if dtype not in _NUMBERS:
        raise TypeError("dtype is %s" % dtype)
    m, k, ldq = _rows("q", q)
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    ctx._chk(hip.lib().dn_i8_restore(ctx.h, m, k, q.data_ptr(), ldq, s.data_ptr(), x.data_ptr(), k, TYPES[dtype], _stream(ctx)), "dn_i8_restore")
    return x


def _weight(ctx, wq, ws, k):
    _check(ctx, "wq", wq, (torch.int8,))
    if wq.dim() != 2 or wq.shape[1] != k:
        raise ValueError("wq has the shape %s, expected [N, %d]" % (tuple(wq.shape), k))
    n, _, ldw = _rows("wq", wq)
    _check(ctx, "ws", ws, (torch.float32,), (n,))
    _vector("ws", ws)
    return n, ldw


def linear(ctx, x, wq, ws, sx=None, bias=None, residual=None, relu=False, out_dtype=None, save=False):
    _check(ctx, "x", x, _NUMBERS + (torch.int8,))
    given = x.dtype == torch.int8
    if given != (sx is not None):
        raise ValueError("sx goes with int8 rows and with nothing else")
    m, k, ldx = _rows("x", x)
    n, ldw = _weight(ctx, wq, ws, k)
    out_dtype = out_dtype or (torch.bfloat16 if given else x.dtype)
    if out_dtype not in _NUMBERS:
        raise TypeError("out_dtype is %s" % out_dtype)
    d = hip.I8Linear(m=m, n=n, k=k, x=x.data_ptr(), ldx=ldx, w=wq.data_ptr(), ldw=ldw, sw=ws.data_ptr(), x_type=TYPES[x.dtype],
                     y_type=TYPES[out_dtype], relu=int(bool(relu)))
    lead = x.shape[:-1]
    if given:
        _check(ctx, "sx", sx, (torch.float32,), lead)
        _vector("sx", sx)
        d.sx = sx.data_ptr()
    if bias is not None:
        _check(ctx, "bias", bias, (torch.float32,), (n,))
        _vector("bias", bias)
        d.bias = bias.data_ptr()
    y = torch.empty(*lead, n, dtype=out_dtype, device=x.device)
    if residual is not None:
        _check(ctx, "residual", residual, (out_dtype,), y.shape)
        d.residual, d.ldr = residual.data_ptr(), _rows("residual", residual)[2]
    d.y, d.ldy = y.data_ptr(), n
    saved = None
    if save:
        mask = torch.empty(m, (n + 7) // 8, dtype=torch.uint8, device=x.device) if relu else None
        if mask is not None:
            d.mask, d.ldmask = mask.data_ptr(), mask.shape[1]
        if given:
            saved = Saved(x, sx, mask)
        else:
            saved = Saved(_empty_rows(x.shape, x.device), torch.empty(lead, dtype=torch.float32, device=x.device), mask)
            d.q, d.ldq, d.s = saved.q.data_ptr(), _pitch(saved.q), saved.s.data_ptr()
    if m:
        _run(ctx, "dn_i8_linear", d)
    return (y, saved) if save else y


def linear_grad(ctx, dy, q, s, wq, ws, mask=None, need_dx=True, need_dw=True, need_db=True, w_dtype=None):
    _check(ctx, "dy", dy, _NUMBERS)
    m, n, ldy = _rows("dy", dy)
    _check(ctx, "q", q, (torch.int8,))
    mq, k, ldq = _rows("q", q)
    if tuple(q.shape[:-1]) != tuple(dy.shape[:-1]):
        raise ValueError("q has the shape %s, dy %s" % (tuple(q.shape), tuple(dy.shape)))
    _check(ctx, "s", s, (torch.float32,), q.shape[:-1])
    _vector("s", s)
    nw, ldw = _weight(ctx, wq, ws, k)
    if nw != n:
        raise ValueError("wq has %d output channels, dy %d" % (nw, n))
    w_dtype = w_dtype or dy.dtype
    if w_dtype not in _NUMBERS:
        raise TypeError("w_dtype is %s" % w_dtype)
    d = hip.I8Grad(m=m, n=n, k=k, dy=dy.data_ptr(), ldy=ldy, q=q.data_ptr(), ldq=ldq, s=s.data_ptr(), w=wq.data_ptr(), ldw=ldw, sw=ws.data_ptr(),
                   dy_type=TYPES[dy.dtype], dw_type=TYPES[w_dtype])
    if mask is not None:
        _check(ctx, "mask", mask, (torch.uint8,), (m, (n + 7) // 8))
        d.mask, d.ldmask = mask.data_ptr(), _rows("mask", mask)[2]
    dx = dw = db = None
    if need_dx:
        dx = torch.empty(*dy.shape[:-1], k, dtype=dy.dtype, device=dy.device)
        d.dx, d.ldx = dx.data_ptr(), k
    if need_dw:
        dw = torch.empty(n, k, dtype=w_dtype, device=dy.device)
        d.dw, d.lddw = dw.data_ptr(), k
    if need_db:
        db = torch.empty(n, dtype=w_dtype, device=dy.device)
        d.db = db.data_ptr()
    if need_dw or need_db or (need_dx and m):
        _run(ctx, "dn_i8_linear_grad", d)
    return dx, dw, db
