"""8-bit dense layers on torch tensors: the checks and allocations behind hip.Context.i8_*, and the layer that is trained with them.

A dense layer y = act(x W^T + b) over rows of x (positions of reads).  Its input and its weight are kept as rows of 8-bit integers with one fp32
scale each (include/dnascent_hip.h has the formulas); the same 8-bit rows are what the product multiplies and what its gradient needs, so a layer that
is being fitted keeps K + 4 bytes per row between forward and backward pass, and one bit per output if a ReLU follows, instead of numbers.
The reference has no counterpart: its network is a frozen SavedModel (tensor.cpp:12-106), trained outside it.

(The wrappers are written for short calls: a small layer's kernel takes a few microseconds, as much as a handful of Python attribute look-ups.)
"""
import copy
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import hip

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}      # DN_T_*
_NUMBERS = (torch.float32, torch.float16, torch.bfloat16)
_F32, _I8, _U8 = torch.float32, torch.int8, torch.uint8
# torch.cuda.current_stream() builds a Stream object; this is the handle alone
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


class Saved(NamedTuple):
    """what a layer keeps for its gradient: q [..., K] int8, s [...] fp32, and mask [rows, (N + 7) // 8] uint8 (bit n % 8 of byte n // 8) or None"""
    q: torch.Tensor
    s: torch.Tensor
    mask: Optional[torch.Tensor]


def _check(ctx, name, t, dtypes, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: a torch tensor is expected, not %s" % (name, type(t).__name__))
    if t.get_device() != ctx.device:                       # -1: not on a GPU
        raise ValueError("%s is on %s, the context on device %d" % (name, t.device, ctx.device))
    if t.dtype not in dtypes:
        raise TypeError("%s is %s" % (name, t.dtype))
    if shape is not None and t.shape != shape:
        raise ValueError("%s has the shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _vector(ctx, name, t, shape):
    """fp32, without gaps; its address"""
    _check(ctx, name, t, (_F32,), shape)
    if not t.is_contiguous():
        raise ValueError("%s is not contiguous" % name)
    return t.data_ptr()


def _rows(name, t):
    """t [..., C] as (rows, C, pitch in elements): its elements stay where they are"""
    shape, stride = t.shape, t.stride()
    if len(shape) == 2 and shape[0] > 1 and shape[1] > 1 and stride[1] == 1 and stride[0] >= shape[1]:
        return shape[0], shape[1], stride[0]
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError("%s has the shape %s: rows of at least one element are expected" % (name, tuple(shape)))
    c = shape[-1]
    if c > 1 and stride[-1] != 1:
        raise ValueError("%s: the elements of a row are not next to each other (call .contiguous())" % name)
    m = t.numel() // c
    lead = [(n, st) for n, st in zip(shape[:-1], stride[:-1]) if n > 1]
    if m <= 1 or not lead:
        return m, c, c
    for (_, outer), (n, inner) in zip(lead[:-1], lead[1:]):
        if outer != n * inner:
            raise ValueError("%s: its rows do not lie at one pitch (call .contiguous())" % name)
    pitch = lead[-1][1]
    if 0 < pitch < c:
        raise ValueError("%s: its rows overlap (call .contiguous())" % name)
    return m, c, pitch


def _empty_rows(shape, device):
    """int8 [..., K] whose rows start at multiples of 16 bytes, and their pitch"""
    k = shape[-1]
    pitch = (k + 15) // 16 * 16
    if pitch == k:
        return torch.empty(shape, dtype=_I8, device=device), k
    return torch.empty(*shape[:-1], pitch, dtype=_I8, device=device)[..., :k], pitch


def _run(ctx, entry, desc):
    lib = hip.lib()
    need = C.c_uint64(0)
    rc = getattr(lib, entry + "_workspace")(ctx.h, desc, need)
    if rc:
        ctx._chk(rc, entry)
    need = need.value
    if need:
        ws = torch.empty(need, dtype=_U8, device=ctx.device)                # torch's allocator: the caller's stream, or the graph being captured, owns it
        rc = getattr(lib, entry)(ctx.h, desc, ws.data_ptr(), need, _stream(ctx.device))
    else:
        rc = getattr(lib, entry)(ctx.h, desc, None, 0, _stream(ctx.device))
    if rc:
        ctx._chk(rc, entry)


def _no_gradient(**tensors):
    """the calls give tensors without a history: one that asks for a gradient would lose it without a word"""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if getattr(t, "requires_grad", False):          # (what is no tensor is refused for that)
                raise ValueError("%s requires a gradient, which this call does not pass on: use dense8.Dense, torch.no_grad() or .detach()" % name)


def rows(ctx, x):
    _check(ctx, "x", x, _NUMBERS)
    m, k, ldx = _rows("x", x)
    q, ldq = _empty_rows(x.shape, x.device)
    s = torch.empty(x.shape[:-1], dtype=_F32, device=x.device)
    rc = hip.lib().dn_i8_rows(ctx.h, m, k, x.data_ptr(), ldx, TYPES[x.dtype], q.data_ptr(), ldq, s.data_ptr(), _stream(ctx.device))
    if rc:
        ctx._chk(rc, "dn_i8_rows")
    return q, s


def restore(ctx, q, s, dtype):
    _check(ctx, "q", q, (_I8,))
    if dtype not in _NUMBERS:
        raise TypeError("dtype is %s" % dtype)
    m, k, ldq = _rows("q", q)
    at = _vector(ctx, "s", s, q.shape[:-1])
    _no_gradient(s=s)
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    rc = hip.lib().dn_i8_restore(ctx.h, m, k, q.data_ptr(), ldq, at, x.data_ptr(), k, TYPES[dtype], _stream(ctx.device))
    if rc:
        ctx._chk(rc, "dn_i8_restore")
    return x


def _weight(ctx, wq, ws, k):
    _check(ctx, "wq", wq, (_I8,))
    if wq.dim() != 2 or wq.shape[1] != k:
        raise ValueError("wq has the shape %s, expected [N, %d]" % (tuple(wq.shape), k))
    n, _, ldw = _rows("wq", wq)
    return n, ldw, _vector(ctx, "ws", ws, (n,))


def linear(ctx, x, wq, ws, sx=None, bias=None, residual=None, relu=False, out_dtype=None, save=False):
    _check(ctx, "x", x, _NUMBERS + (_I8,))
    given = x.dtype is _I8
    if given != (sx is not None):
        raise ValueError("sx goes with int8 rows and with nothing else")
    m, k, ldx = _rows("x", x)
    n, ldw, at_ws = _weight(ctx, wq, ws, k)
    out_dtype = out_dtype or (torch.bfloat16 if given else x.dtype)
    if out_dtype not in _NUMBERS:
        raise TypeError("out_dtype is %s" % out_dtype)
    _no_gradient(x=x, ws=ws, sx=sx, bias=bias, residual=residual)
    lead = x.shape[:-1]
    at_sx = _vector(ctx, "sx", sx, lead) if given else 0
    at_bias = _vector(ctx, "bias", bias, (n,)) if bias is not None else 0
    y = torch.empty(lead + (n,), dtype=out_dtype, device=x.device)
    at_res = ldr = 0
    if residual is not None:
        _check(ctx, "residual", residual, (out_dtype,), y.shape)
        at_res, ldr = residual.data_ptr(), _rows("residual", residual)[2]
    saved = None
    at_mask = ldmask = at_q = ldq = at_s = 0
    if save:
        mask = None
        if relu:
            ldmask = (n + 7) // 8
            mask = torch.empty(m, ldmask, dtype=_U8, device=x.device)
            at_mask = mask.data_ptr()
        if given:
            saved = Saved(x, sx, mask)
        else:
            q, ldq = _empty_rows(x.shape, x.device)
            saved = Saved(q, torch.empty(lead, dtype=_F32, device=x.device), mask)
            at_q, at_s = q.data_ptr(), saved.s.data_ptr()
    if m:
        _run(ctx, "dn_i8_linear", hip.I8_LINEAR.pack(m, n, k, x.data_ptr(), ldx, at_sx, wq.data_ptr(), ldw, at_ws, at_bias, at_res, ldr, y.data_ptr(), n,
                                                     at_mask, ldmask, at_q, ldq, at_s, TYPES[x.dtype], TYPES[out_dtype], 1 if relu else 0, 0))
    return (y, saved) if save else y


def linear_grad(ctx, dy, q, s, wq, ws, mask=None, need_dx=True, need_dw=True, need_db=True, w_dtype=None):
    _check(ctx, "dy", dy, _NUMBERS)
    m, n, ldy = _rows("dy", dy)
    _check(ctx, "q", q, (_I8,))
    mq, k, ldq = _rows("q", q)
    lead = dy.shape[:-1]
    if q.shape[:-1] != lead:
        raise ValueError("q has the shape %s, dy %s" % (tuple(q.shape), tuple(dy.shape)))
    at_s = _vector(ctx, "s", s, lead)
    nw, ldw, at_ws = _weight(ctx, wq, ws, k)
    if nw != n:
        raise ValueError("wq has %d output channels, dy %d" % (nw, n))
    _no_gradient(dy=dy, s=s, ws=ws)
    w_dtype = w_dtype or dy.dtype
    if w_dtype not in _NUMBERS:
        raise TypeError("w_dtype is %s" % w_dtype)
    at_mask = ldmask = at_dx = at_dw = at_db = 0
    if mask is not None:
        _check(ctx, "mask", mask, (_U8,), (m, (n + 7) // 8))
        at_mask, ldmask = mask.data_ptr(), _rows("mask", mask)[2]
    dx = dw = db = None
    if need_dx:
        dx = torch.empty(q.shape, dtype=dy.dtype, device=dy.device)
        at_dx = dx.data_ptr()
    if need_dw:
        dw = torch.empty(n, k, dtype=w_dtype, device=dy.device)
        at_dw = dw.data_ptr()
    if need_db:
        db = torch.empty(n, dtype=w_dtype, device=dy.device)
        at_db = db.data_ptr()
    if need_dw or need_db or (need_dx and m):
        _run(ctx, "dn_i8_linear_grad", hip.I8_GRAD.pack(m, n, k, dy.data_ptr(), ldy, at_mask, ldmask, q.data_ptr(), ldq, at_s, wq.data_ptr(), ldw, at_ws,
                                                        at_dx, k, at_dw, k, at_db, TYPES[dy.dtype], TYPES[w_dtype]))
    return dx, dw, db


# ---- the layer that is trained with them ----------------------------------------------------------------------------------------------------------------
def _packed(t):
    """t, or a copy without gaps if its rows do not lie at one pitch (the gradient of a sum is one number repeated, for instance)"""
    try:
        _rows("", t)
        return t
    except ValueError:
        return t.contiguous()


def _dense(ctx, x, weight, bias, residual, relu, save):
    """the layer's product: (what linear returns, the weight's rows, their scales)"""
    wq, ws = rows(ctx, _packed(weight))
    return linear(ctx, _packed(x), wq, ws, bias=None if bias is None else bias.float(), residual=None if residual is None else _packed(residual), relu=relu, save=save), wq, ws


class _Layer(torch.autograd.Function):
    """The forward pass keeps what i8_linear saves and the weight's 8-bit rows; both quantisers count as the identity in the backward pass, so the gradients
    are those of the product that was computed."""

    @staticmethod
    def forward(fn, x, weight, bias, residual, ctx, relu):
        (y, saved), wq, ws = _dense(ctx, x, weight, bias, residual, relu, True)
        fn.save_for_backward(saved.q, saved.s, saved.mask, wq, ws)
        fn.ctx, fn.w_dtype, fn.b_dtype = ctx, weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(fn, dy):
        q, s, mask, wq, ws = fn.saved_tensors
        need_x, need_w, need_b, need_r = fn.needs_input_grad[:4]
        dr = None
        if need_r:
            dr = dy
            if mask is not None:
                bits = torch.arange(dy.shape[-1], device=dy.device)
                keep = mask[:, bits >> 3].bitwise_right_shift((bits & 7).to(_U8)).bitwise_and(1).bool()
                dr = torch.where(keep.view(dy.shape), dy, torch.zeros((), dtype=dy.dtype, device=dy.device))
        dx, dw, db = linear_grad(fn.ctx, _packed(dy), q, s, wq, ws, mask, need_x, need_w, need_b, fn.w_dtype)
        return dx, dw, db if db is None else db.to(fn.b_dtype), dr, None, None


class Dense(torch.nn.Module):
    """y [..., N] = act(x W^T + b (+ residual)) whose forward pass multiplies 8-bit rows and whose backward pass reads them again: weight [N, K] and bias [N] are
    parameters (fp32, fp16 or bf16) on ctx's device; x [..., K] of the same types.  Between the passes a row of x costs K + 4 bytes, without gradients nothing.

    A pass can be captured into a graph like any of torch's (its workspaces are torch tensors); as with those, no eager graph over the same parameters
    may be alive while a backward pass is being captured.

    A pointwise convolution of a model description (cnn_model.py: an op "conv" with k = 1) is such a layer over positions: from_op() reads it, store() writes it
    back, so that a description can be fitted here and run by Context.load_cnn."""

    def __init__(self, ctx, k, n, bias=True, relu=False, dtype=torch.float32):
        super().__init__()
        if dtype not in _NUMBERS:
            raise TypeError("dtype is %s" % dtype)
        device = torch.device("cuda", ctx.device)
        self.ctx, self.relu = ctx, bool(relu)
        self.weight = torch.nn.Parameter((torch.randn(n, k, device=device) * k ** -0.5).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=device)) if bias else None

    def __deepcopy__(self, memo):
        memo[id(self.ctx)] = self.ctx                      # parameters of its own, the same device context
        new = type(self).__new__(type(self))
        memo[id(self)] = new
        new.__dict__.update(copy.deepcopy(self.__dict__, memo))
        return new

    def forward(self, x, residual=None):
        if not (torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in (x, self.weight, self.bias, residual))):
            return _dense(self.ctx, x, self.weight, self.bias, residual, self.relu, False)[0]           # nothing to keep
        return _Layer.apply(x, self.weight, self.bias, residual, self.ctx, self.relu)

    @staticmethod
    def _op(desc, i):
        op = desc["ops"][i]
        if op["op"] != "conv" or op["k"] != 1:
            raise ValueError("op %d is no pointwise convolution" % i)
        return op, op["cin"], op["cout"]

    @classmethod
    def from_op(cls, ctx, desc, blob, i, dtype=torch.float32):
        """op i of a description: W = kernel^T times the folded BatchNorm's factor, b = its shift.  An op that adds a buffer (add >= 0) takes it as `residual`."""
        op, k, n = cls._op(desc, i)
        w = torch.from_numpy(blob[op["w"]:op["w"] + k * n].reshape(k, n).copy()).t() * torch.from_numpy(blob[op["scale"]:op["scale"] + n].copy())[:, None]
        layer = cls(ctx, k, n, relu=op["relu"], dtype=dtype)
        with torch.no_grad():
            layer.weight.copy_(w)
            layer.bias.copy_(torch.from_numpy(blob[op["shift"]:op["shift"] + n].copy()))
        return layer

    def store(self, desc, blob, i):
        """the parameters into op i of the description's blob, in place: the kernel holds W^T, the factor becomes one"""
        op, k, n = self._op(desc, i)
        if (n, k) != tuple(self.weight.shape) or op["relu"] != self.relu:
            raise ValueError("op %d has another shape or activation than this layer" % i)
        blob[op["w"]:op["w"] + k * n] = self.weight.detach().float().t().reshape(-1).cpu().numpy()
        blob[op["scale"]:op["scale"] + n] = 1.0
        blob[op["shift"]:op["shift"] + n] = 0.0 if self.bias is None else self.bias.detach().float().cpu().numpy()
