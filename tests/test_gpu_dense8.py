"""GPU: the 8-bit dense layers against plain implementations in 64 bits, through hip.Context.i8_*.

Tolerances (u = half a step of the output type relative to the value: fp32 2^-24, fp16 2^-11, bf16 2^-8; T = the sum of the magnitudes of an output's terms):
  rows      bits: every operation is defined in fp32
  restore   u |q s|, and 2^-24 of it where the product passes through fp32
  linear    the integer sum is exact; its conversion, two products and up to two additions round in fp32, each by at most 2^-24 of a value that
            T bounds, then one rounding to the type: u |y| + 6 2^-24 T
  gradient  the factor that carries the scale is held in one fp16 piece (at most 2^-11 of the value: a rounding of the product to fp32, one to fp16)
            for 16-bit results and two (2^-21) for fp32 results; the sums are fp32, in at most M (or N) additions of at most 2^-24 T each:
            u |g| + (2^-11 or 2^-21 + terms 2^-24) T
The smallest numbers of fp16 add 2^-25 (half its smallest step) everywhere."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from dnascent_amd import hip

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}
# one row, one element, odd and even sizes on both sides of 16, 64, 128 and 256, long rows, many rows
SHAPES = [(1, 1, 1), (1, 256, 256), (3, 17, 5), (16, 64, 64), (17, 33, 100), (64, 128, 128), (65, 129, 127), (200, 64, 64), (257, 256, 256), (511, 64, 256),
          (1000, 131, 77), (130, 1000, 1029), (13, 1000, 4352), (1, 4096, 1024), (33, 40, 4353), (4097, 256, 128), (5000, 8, 16), (700, 520, 384)]


@pytest.fixture(scope="module")
def ctx():
    c = hip.Context(0)
    yield c
    c.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def some_rows(m, k, dtype, seed):
    g = gen(seed)
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    if m > 2:
        x[1] = 0                                           # a row of zeros
    return x.to(dtype)


def codes(x):
    """the definition, in numpy's fp32: q as int64, s as fp32"""
    x = x.detach().float().cpu().numpy()
    with np.errstate(all="ignore"):
        a = np.abs(x).max(1)                               # NaN stays NaN
        live = np.isfinite(a) & (a >= np.float32(2.0 ** -120))
        r = np.where(live, np.float32(127) / np.where(live, a, np.float32(1)), np.float32(0)).astype(np.float32)
        s = np.where(live, a / np.float32(127), np.where(np.isfinite(a), np.float32(0), np.float32("nan"))).astype(np.float32)
        q = np.where(live[:, None], np.rint(x * r[:, None]), 0)
    return q.astype(np.int64), s


def bits(mask, n):
    return ((mask.cpu().unsqueeze(2).int() >> torch.arange(8)) & 1).reshape(mask.shape[0], -1)[:, :n].bool()


def within(got, want, terms, dtype, u):
    got, want, terms = got.double().cpu(), want.double().cpu(), terms.double().cpu()
    off = (got - want).abs()
    room = HALF[dtype] * want.abs() + u * terms + TINY[dtype]
    over = want.abs() - room > torch.finfo(dtype).max      # behind the type's largest number there is only infinity
    assert (got[over] == want[over].sign() * math.inf).all()
    off[over] = 0
    bad = ~(off <= room)
    assert not bad.any(), "%d of %d outside, worst %.3g of its room" % (int(bad.sum()), bad.numel(), float((off / room).max()))


def eight(n, k, seed):
    g = gen(seed)
    wq = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    return wq, torch.rand(n, generator=g, device="cuda") * 0.01 + 0.001


def linear_ref(q, s, wq, ws, bias=None, residual=None):
    """(y, T) in 64 bits before act and rounding"""
    q, wq = torch.as_tensor(q).double().cpu(), wq.double().cpu()
    s, ws = torch.as_tensor(s).double().cpu(), ws.double().cpu()
    y = (q @ wq.t()) * s[:, None] * ws
    t = y.abs()
    if bias is not None:
        y, t = y + bias.double().cpu(), t + bias.double().abs().cpu()
    if residual is not None:
        y, t = y + residual.double().cpu(), t + residual.double().abs().cpu()
    return y, t


# ---- rows in 8 bits ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,k", sorted({(m, k) for m, _, k in SHAPES} | {(1, 64), (5, 15), (3, 8193), (70000, 3)}))
def test_rows_and_restore(ctx, m, k, dtype):
    x = some_rows(m, k, dtype, 1000 * m + k)
    q, s = ctx.i8_rows(x)
    qr, sr = codes(x)
    assert q.shape == x.shape and np.array_equal(q.cpu().numpy(), qr) and s.cpu().numpy().tobytes() == sr.tobytes()
    for out in (F32, F16, BF16):
        y = ctx.i8_restore(q, s, out)
        want = torch.from_numpy(qr).double() * torch.from_numpy(sr).double()[:, None]
        within(y, want, want.abs(), out, 2.0 ** -24)       # straight to the type, or through fp32 (half a step of that more)


def test_rows_with_nothing_in_them_or_too_much(ctx):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(12, 100, device="cuda")
    x[0] = 0
    x[1] = 2.0 ** -121
    x[2] = 2.0 ** -120
    x[3, 7] = nan
    x[4, 99] = inf
    x[5, 0] = -inf
    x[6] = -0.0
    x[7] = torch.finfo(F32).max
    x[8] = torch.finfo(F32).min
    x[9] = nan
    x[10] *= 2.0 ** -126
    q, s = ctx.i8_rows(x)
    qr, sr = codes(x)
    assert np.array_equal(q.cpu().numpy(), qr) and np.array_equal(s.cpu().numpy(), sr, equal_nan=True)
    wq, ws = eight(33, 100, 5)
    y = ctx.i8_linear(x, wq, ws)
    bad = torch.tensor([3, 4, 5, 9])
    ok = torch.tensor([i for i in range(12) if i not in (3, 4, 5, 9)])
    assert y.cpu()[bad].isnan().all()
    want, t = linear_ref(qr[ok], sr[ok], wq, ws)
    within(y.cpu()[ok], want, t, F32, 6 * 2.0 ** -24)
    y, saved = ctx.i8_linear(x, wq, ws, relu=True, save=True)             # NaN passes a ReLU, and its bit is clear (a NaN is not > 0)
    assert y.cpu()[bad].isnan().all() and not bits(saved.mask, 33)[bad].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_at_borders_round_to_even(ctx, dtype):
    k = 256
    x = torch.full((4, k), 127.0)
    x[:, 1:] = torch.arange(k - 1) / 2.0 - 63.5            # with a = 127, r = 1: halves are ties
    q, s = ctx.i8_rows(x.to(dtype).cuda())
    assert np.array_equal(q.cpu().numpy(), np.rint(x.to(dtype).float().numpy()).astype(np.int8)) and (s.cpu() == 1).all()


# ---- the product ----------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F32, F16)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(ctx, m, n, k, dtype, out):
    x = some_rows(m, k, dtype, m + n + k)
    wq, ws = eight(n, k, 7 * m + n)
    bias = torch.randn(n, generator=gen(3), device="cuda")
    y = ctx.i8_linear(x, wq, ws, bias=bias, out_dtype=out)
    want, t = linear_ref(*codes(x), wq, ws, bias)
    assert y.shape == (m, n) and y.dtype == out
    within(y, want, t, out, 6 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_of_given_rows_relu_residual_saved(ctx, m, n, k, dtype):
    """everything at once; then the same layer from numbers, which saves the rows that it multiplied"""
    x = some_rows(m, k, dtype, m + n + k + 1)
    wq, ws = eight(n, k, 5 * m + n)
    bias = torch.randn(n, generator=gen(4), device="cuda")
    res = torch.randn(m, n, generator=gen(5), device="cuda").to(dtype)
    qr, sr = codes(x)
    q = torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    q[:, k:] = 99                                          # what lies behind a row's end is not read as part of it
    q = q[:, :k]
    q.copy_(torch.from_numpy(qr))
    s = torch.from_numpy(sr).cuda()
    want, t = linear_ref(qr, sr, wq, ws, bias, res)
    y, saved = ctx.i8_linear(q, wq, ws, sx=s, bias=bias, residual=res, relu=True, out_dtype=dtype, save=True)
    within(y, want.clamp(min=0), t, dtype, 6 * 2.0 ** -24)
    sure = want.abs() > 6 * 2.0 ** -24 * t
    assert torch.equal(bits(saved.mask, n)[sure], (want > 0)[sure])
    y2, saved2 = ctx.i8_linear(x, wq, ws, bias=bias, residual=res, relu=True, out_dtype=dtype, save=True)
    assert torch.equal(y, y2) and torch.equal(saved.mask, saved2.mask)
    assert np.array_equal(saved2.q.cpu().numpy(), qr) and saved2.s.cpu().numpy().tobytes() == sr.tobytes()
    if n % 8:
        assert not (saved.mask[:, -1].cpu() >> (n % 8)).any()             # the bits behind the last output are clear


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_reads_strided_unaligned_and_broadcast_rows(ctx, m):
    n, k = 70, 90
    big = some_rows(m * 3, 200, F16, m)
    wq, ws = eight(n, k, 9)
    odd = torch.zeros(n * k + 1, dtype=torch.int8, device="cuda")[1:].view(n, k)      # rows at no boundary at all
    odd.copy_(wq)
    wide = torch.randint(-127, 128, (n, 131), device="cuda", dtype=torch.int8)[:, 3:3 + k]
    wide.copy_(wq)
    for x in (big[::3, 7:7 + k], big[:m, :k], big[:1, 1:1 + k].expand(m, k)):
        want, t = linear_ref(*codes(x), wq, ws)
        for w in (wq, odd, wide):
            within(ctx.i8_linear(x, w, ws), want, t, F16, 6 * 2.0 ** -24)
    q, s = (torch.as_tensor(v) for v in codes(big[:m, :k]))
    qu = torch.zeros(m * k + 3, dtype=torch.int8, device="cuda")[3:].view(m, k)
    qu.copy_(q)
    want, t = linear_ref(q, s, wq, ws)
    for w in (wq, odd, wide):
        within(ctx.i8_linear(qu, w, ws, sx=s.cuda(), out_dtype=F32), want, t, F32, 6 * 2.0 ** -24)


def test_linear_with_the_lowest_code(ctx):
    """-128 is no code that i8_rows writes, but a caller's rows may hold it: the integer sums stay inside 32 bits up to the largest K"""
    k = 131071
    q = torch.full((2, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
    w = torch.full((3, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
    one = torch.ones(3, device="cuda")
    y = ctx.i8_linear(q, w, one, sx=one[:2].contiguous(), out_dtype=F32)
    assert (y == float(np.float32(128 * 128 * k))).all()


def test_leading_dimensions_and_no_rows(ctx):
    wq, ws = eight(24, 40, 11)
    x = some_rows(30, 40, BF16, 12)
    flat = ctx.i8_linear(x, wq, ws, relu=True)
    y, saved = ctx.i8_linear(x.view(2, 3, 5, 40), wq, ws, relu=True, save=True)
    assert y.shape == (2, 3, 5, 24) and torch.equal(y.view(30, 24), flat) and saved.q.shape == (2, 3, 5, 40) and saved.s.shape == (2, 3, 5)
    dy = some_rows(30, 24, BF16, 13)
    a = ctx.i8_linear_grad(dy.view(2, 3, 5, 24), saved.q, saved.s, wq, ws, mask=saved.mask)
    b = ctx.i8_linear_grad(dy, saved.q.reshape(30, 40), saved.s.view(30), wq, ws, mask=saved.mask)
    assert a[0].shape == (2, 3, 5, 40) and torch.equal(a[0].view(30, 40), b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    assert torch.equal(ctx.i8_linear(x[0], wq, ws), ctx.i8_linear(x[:1], wq, ws)[0])
    none = x[:0]
    q, s = ctx.i8_rows(none)
    assert q.shape == (0, 40) and s.shape == (0,) and ctx.i8_restore(q, s, F32).shape == (0, 40)
    y, saved = ctx.i8_linear(none, wq, ws, relu=True, save=True)
    assert y.shape == (0, 24) and saved.mask.shape == (0, 3)
    dx, dw, db = ctx.i8_linear_grad(dy[:0], q, s, wq, ws, mask=saved.mask)
    assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (24, 40)


# ---- the gradient ---------------------------------------------------------------------------------------------------------------------------------------
def grad_case(m, n, k, dtype, seed, relu):
    g = gen(seed)
    q, s = eight(m, k, seed + 1)
    wq, ws = eight(n, k, seed + 2)
    dy = (torch.randn(m, n, generator=g, device="cuda") * 1e-3 * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))).to(dtype)
    mask = torch.randint(0, 256, (m, (n + 7) // 8), generator=g, device="cuda", dtype=torch.uint8) if relu else None
    return dy, q, s, wq, ws, mask


def grad_ref(dy, q, s, wq, ws, mask):
    dz = dy.double().cpu()
    if mask is not None:
        dz = torch.where(bits(mask, dy.shape[1]), dz, torch.zeros_like(dz))
    xh = q.double().cpu() * s.double().cpu()[:, None]
    wh = wq.double().cpu() * ws.double().cpu()[:, None]
    return (dz @ wh, dz.t() @ xh, dz.sum(0)), (dz.abs() @ wh.abs(), dz.abs().t() @ xh.abs(), dz.abs().sum(0))


def check_grad(got, ref, m, n, dtype, w_dtype):
    (dx, dw, db), (tx, tw, tb) = ref
    piece = lambda t: 2.0 ** -21 if t == F32 else 2.0 ** -11  # noqa: E731
    within(got[0], dx, tx, dtype, piece(dtype) + n * 2.0 ** -24)
    within(got[1], dw, tw, w_dtype, piece(w_dtype) + m * 2.0 ** -24)
    within(got[2], db, tb, w_dtype, m * 2.0 ** -24)


@pytest.mark.parametrize("dtype,w_dtype,relu", [(F32, F32, True), (F16, F16, False), (BF16, BF16, True), (BF16, F32, False), (F32, BF16, True)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_grad(ctx, m, n, k, dtype, w_dtype, relu):
    case = grad_case(m, n, k, dtype, m + 3 * n + k, relu)
    got = ctx.i8_linear_grad(*case[:5], mask=case[5], w_dtype=w_dtype)
    assert [t.dtype for t in got] == [dtype, w_dtype, w_dtype]
    check_grad(got, grad_ref(*case), m, n, dtype, w_dtype)
    again = ctx.i8_linear_grad(*case[:5], mask=case[5], w_dtype=w_dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, again))             # the order of every sum is fixed
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False)):
        part = ctx.i8_linear_grad(*case[:5], mask=case[5], w_dtype=w_dtype, need_dx=need[0], need_dw=need[1], need_db=need[2])
        for want, p, full in zip(need, part, got):
            assert (p is not None) == want and (p is None or torch.equal(p, full))


@pytest.mark.parametrize("m,n,k", [(40, 33, 50), (700, 256, 256), (600, 300, 520)])
def test_grad_of_strided_unaligned_and_broadcast_tensors(ctx, m, n, k):
    dy, q, s, wq, ws, mask = grad_case(m, n, k, BF16, 77, True)
    ref = grad_ref(dy, q, s, wq, ws, mask)
    wide = torch.zeros(m, n + 9, dtype=BF16, device="cuda")
    wide[:, 3:3 + n] = dy
    qo = torch.zeros(m * (k + 1) + 1, dtype=torch.int8, device="cuda")[1:].view(m, k + 1)[:, :k]
    qo.copy_(q)
    wo = torch.zeros(n * k + 5, dtype=torch.int8, device="cuda")[5:].view(n, k)
    wo.copy_(wq)
    mw = torch.zeros(m, (n + 7) // 8 + 2, dtype=torch.uint8, device="cuda")
    mw[:, 1:-1] = mask
    check_grad(ctx.i8_linear_grad(wide[:, 3:3 + n], qo, s, wo, ws, mask=mw[:, 1:-1]), ref, m, n, BF16, BF16)
    one = dy[:1].expand(m, n)                              # one gradient row for all
    check_grad(ctx.i8_linear_grad(one, q, s, wq, ws, mask=mask), grad_ref(one, q, s, wq, ws, mask), m, n, BF16, BF16)


@pytest.mark.parametrize("m,n,k", [(65, 70, 40), (3000, 128, 256), (900, 520, 384)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_grad_keeps_what_is_not_finite_where_it_belongs(ctx, m, n, k, dtype):
    """NaN and infinity under a cleared bit are dropped; one that is kept reaches its own row of dx and its own output channel of dw and db, nothing else.
    A row that had no 8-bit form (s = NaN) makes dw NaN, as it does in the plain product, and leaves dx alone."""
    dy, q, s, wq, ws, mask = grad_case(m, n, k, dtype, 99, True)
    inf, nan = float("inf"), float("nan")
    keep = bits(mask, n)
    keep[3] = True
    keep[4] = False
    keep[5, 1::2] = False
    keep[5, ::2] = True
    keep[7] = False
    packed = np.packbits(keep.numpy(), axis=1, bitorder="little")
    mask = torch.from_numpy(packed).cuda()
    dy[4] = nan
    dy[5, 1] = inf
    dy[7, 0] = -inf
    dy[3, 2] = nan
    dy[3, 6] = inf
    s[7] = nan                                             # behind dz = 0: 0 * NaN = NaN in dw, as in the plain product
    got = ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask)
    dx, dw, db = (t.cpu() for t in got)
    assert dx[3].isnan().all()                             # NaN and infinity meet in this row
    rows = torch.tensor([i for i in range(m) if i != 3])
    assert dx[rows].isfinite().all()
    assert dw.isnan().all()                                # every channel has row 7's NaN
    assert db[2].isnan() and db[6] == inf and db[[i for i in range(n) if i not in (2, 6)]].isfinite().all()
    s[7] = 0.01
    dx, dw, db = (t.cpu() for t in ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask))
    rest = torch.tensor([i for i in range(n) if i not in (2, 6)])
    assert dw[2].isnan().all() and not dw[6].isfinite().any() and dw[rest].isfinite().all()
    clean = dy.clone()
    clean[4] = 0
    clean[5, 1] = 0
    clean[7, 0] = 0
    clean[3, 2] = 0
    clean[3, 6] = 0
    (rx, rw, rb), (tx, tw, tb) = grad_ref(clean, q, s, wq, ws, mask)
    piece = 2.0 ** -21 if dtype == F32 else 2.0 ** -11
    within(dx[rows], rx[rows], tx[rows], dtype, piece + n * 2.0 ** -24)
    within(dw[rest], rw[rest], tw[rest], dtype, piece + m * 2.0 ** -24)
    within(db[rest], rb[rest], tb[rest], dtype, m * 2.0 ** -24)


@pytest.mark.parametrize("m,n,k", [(300, 64, 64), (2000, 256, 256), (800, 300, 520)])
def test_grad_over_a_wide_range_of_sizes(ctx, m, n, k):
    """rows of gradients from 2^-60 to 2^60, the large ones in the middle and at the end: whatever scale the fp16 pieces take, a result keeps its relative
    accuracy against the sum of its own terms"""
    dy, q, s, wq, ws, mask = grad_case(m, n, k, F32, 5, False)
    e = torch.randint(-60, 1, (m, 1), generator=gen(6), device="cuda").float()
    e[m // 2] = 60
    e[m - 1] = 58
    dy = torch.randn(m, n, generator=gen(7), device="cuda") * torch.exp2(e)
    for dtype in (F32, BF16):
        d = dy.to(dtype)
        check_grad(ctx.i8_linear_grad(d, q, s, wq, ws), grad_ref(d, q, s, wq, ws, None), m, n, dtype, dtype)
    small = (torch.randn(m, n, generator=gen(8), device="cuda") * 2.0 ** -100).to(BF16)
    check_grad(ctx.i8_linear_grad(small, q, s, wq, ws), grad_ref(small, q, s, wq, ws, None), m, n, BF16, BF16)


def test_grad_against_differences(ctx):
    """y is linear in the rows it multiplies: L(q + d) - L(q) for L = sum dy * y equals sum dx * (s d), and the same in the weight's rows and the bias.
    The forward pass in fp32 rounds each y by 4 2^-24 of its terms; L adds m n of them."""
    m, n, k = 37, 29, 45
    dy, q, s, wq, ws, _ = grad_case(m, n, k, F32, 21, False)
    q, wq = q // 2, wq // 2
    bias = torch.randn(n, device="cuda")
    dx, dw, db = (t.double().cpu() for t in ctx.i8_linear_grad(dy, q, s, wq, ws))
    L = lambda q_, w_, b_: (dy.double() * ctx.i8_linear(q_, w_, ws, sx=s, bias=b_, out_dtype=F32).double()).sum().item()  # noqa: E731
    base = L(q, wq, bias)
    room = 12 * 2.0 ** -24 * float((dy.double().abs() * (linear_ref(q.abs(), s, wq.abs(), ws, bias.abs())[1].cuda())).sum())
    for seed in range(4):
        d = torch.randint(-9, 10, (m, k), generator=gen(seed), device="cuda", dtype=torch.int8)
        assert abs(L(q + d, wq, bias) - base - float((dx * d.double().cpu() * s.double().cpu()[:, None]).sum())) <= 2 * room
        d = torch.randint(-9, 10, (n, k), generator=gen(seed + 9), device="cuda", dtype=torch.int8)
        assert abs(L(q, wq + d, bias) - base - float((dw * d.double().cpu() * ws.double().cpu()[:, None]).sum())) <= 2 * room
        d = torch.randn(n, generator=gen(seed + 20), device="cuda")
        assert abs(L(q, wq, bias + d) - base - float((db * d.double().cpu()).sum())) <= 2 * room


# ---- how the calls behave beside each other ---------------------------------------------------------------------------------------------------------------
def _mixed(ctx, m, n, k, dtype, seed):
    """a call of every entry over one layer"""
    x = some_rows(m, k, dtype, seed)
    wq, ws = eight(n, k, seed + 1)
    dy = some_rows(m, n, dtype, seed + 2)

    def call():
        y, saved = ctx.i8_linear(x, wq, ws, relu=True, save=True)
        return (y, saved.q, saved.s, saved.mask, ctx.i8_restore(saved.q, saved.s, dtype)) + ctx.i8_linear_grad(dy, saved.q, saved.s, wq, ws, mask=saved.mask)
    return call


def test_outputs_end_where_they_end(ctx):
    """C level: rows at a pitch, canaries between and behind them"""
    L = hip.lib()
    for m, n, k in ((1, 5, 7), (19, 70, 90), (300, 130, 66), (70, 600, 520), (2100, 200, 250)):
        x = some_rows(m, k, BF16, k)
        wq, ws = eight(n, k, n)
        y = torch.full((m + 2, n + 5), 7.0, dtype=BF16, device="cuda")
        q = torch.full((m + 2, k + 40), 77, dtype=torch.int8, device="cuda")
        s = torch.full((m + 2,), 7.0, device="cuda")
        mask = torch.full((m + 2, (n + 7) // 8 + 3), 0xA5, dtype=torch.uint8, device="cuda")
        d = hip.i8_desc(hip.I8_LINEAR_FIELDS, m=m, n=n, k=k, x=x.data_ptr(), ldx=k, w=wq.data_ptr(), ldw=wq.stride(0), sw=ws.data_ptr(), y=y.data_ptr(), ldy=n + 5,
                         mask=mask.data_ptr(), ldmask=mask.shape[1], q=q.data_ptr(), ldq=k + 40, s=s.data_ptr(), x_type=2, y_type=2, relu=1)
        need = C.c_uint64(0)
        assert L.dn_i8_linear_workspace(ctx.h, d, C.byref(need)) == 0
        ws_ = torch.full((need.value + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        assert L.dn_i8_linear(ctx.h, d, ws_.data_ptr(), need.value, st) == 0
        ref, saved = ctx.i8_linear(x, wq, ws, relu=True, save=True)
        assert torch.equal(y[:m, :n], ref) and (y[:m, n:] == 7).all() and (y[m:] == 7).all()
        assert torch.equal(q[:m, :k], saved.q) and (q[m:] == 77).all() and (q[:m, (k + 15) // 16 * 16:] == 77).all() and not q[:m, k:(k + 15) // 16 * 16].any()
        assert torch.equal(s[:m], saved.s) and (s[m:] == 7).all()
        assert torch.equal(mask[:m, :-3], saved.mask) and (mask[:m, -3:] == 0xA5).all() and (mask[m:] == 0xA5).all()
        assert (ws_[need.value:] == 0xA5).all()
        dy = some_rows(m, n, BF16, 3)
        dx = torch.full((m + 2, k + 3), 7.0, dtype=BF16, device="cuda")
        dw = torch.full((n + 2, k + 3), 7.0, device="cuda")
        db = torch.full((n + 2,), 7.0, device="cuda")
        g = hip.i8_desc(hip.I8_GRAD_FIELDS, m=m, n=n, k=k, dy=dy.data_ptr(), ldy=n, mask=mask.data_ptr(), ldmask=mask.shape[1], q=q.data_ptr(), ldq=k + 40, s=s.data_ptr(),
                       w=wq.data_ptr(), ldw=wq.stride(0), sw=ws.data_ptr(), dx=dx.data_ptr(), ldx=k + 3, dw=dw.data_ptr(), lddw=k + 3, db=db.data_ptr(), dy_type=2, dw_type=0)
        assert L.dn_i8_linear_grad_workspace(ctx.h, g, C.byref(need)) == 0
        ws_ = torch.full((need.value + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        assert L.dn_i8_linear_grad(ctx.h, g, ws_.data_ptr(), need.value, st) == 0
        rx, rw, rb = ctx.i8_linear_grad(dy, saved.q, saved.s, wq, ws, mask=saved.mask, w_dtype=F32)
        assert torch.equal(dx[:m, :k], rx) and (dx[:m, k:] == 7).all() and (dx[m:] == 7).all()
        assert torch.equal(dw[:n, :k], rw) and (dw[:n, k:] == 7).all() and (dw[n:] == 7).all()
        assert torch.equal(db[:n], rb) and (db[n:] == 7).all() and (ws_[need.value:] == 0xA5).all()
        if need.value:
            assert L.dn_i8_linear_grad(ctx.h, g, ws_.data_ptr(), need.value - 1, st) == -3
            assert L.dn_i8_linear_grad(ctx.h, g, ws_.data_ptr() + 8, need.value, st) == -3
            assert b"workspace" in L.dn_last_error(ctx.h)


@pytest.mark.parametrize("m,n,k", [(1, 256, 256), (13, 1000, 1029), (3000, 256, 256), (600, 520, 384)])
def test_captured_calls_replay(ctx, m, n, k):
    """two graphs of the same layer (each with its own workspace), replayed in turn with eager calls between, new inputs each time"""
    calls = [_mixed(ctx, m, n, k, BF16, 31), _mixed(ctx, m, n, k, F32, 32)]
    graphs = []
    for call in calls:
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            call()
        torch.cuda.current_stream().wait_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    want = [call() for call in calls]
    for rep in range(4):
        for (g, out), w in zip(graphs, want):
            for t in out:
                t.zero_()
            g.replay()
            eager = calls[rep % 2]()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w)), rep
            assert all(torch.equal(a, b) for a, b in zip(eager, want[rep % 2]))


def test_two_streams_at_once(ctx):
    calls = [_mixed(ctx, 4000, 256, 256, BF16, 41), _mixed(ctx, 900, 520, 384, F16, 42)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for st, call, g in zip(streams, calls, got):
            with torch.cuda.stream(st):
                g.append(call())
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for out in g for a, b in zip(out, w))


def test_refusals(ctx):
    x = some_rows(6, 32, BF16, 1)
    wq, ws = eight(8, 32, 2)
    q, s = ctx.i8_rows(x)
    dy = some_rows(6, 8, BF16, 3)
    for call, kind in [(lambda: ctx.i8_rows(x.cpu()), ValueError), (lambda: ctx.i8_rows(x.double()), TypeError), (lambda: ctx.i8_rows(x.t()), ValueError),
                       (lambda: ctx.i8_restore(q, s[:3], F32), ValueError), (lambda: ctx.i8_restore(q, s, torch.int8), TypeError),
                       (lambda: ctx.i8_linear(x, wq[:, :31], ws), ValueError), (lambda: ctx.i8_linear(x, wq, ws[:7]), ValueError),
                       (lambda: ctx.i8_linear(x, wq, ws.double()), TypeError), (lambda: ctx.i8_linear(x, wq, ws, sx=s), ValueError),
                       (lambda: ctx.i8_linear(q, wq, ws), ValueError), (lambda: ctx.i8_linear(x, wq, ws, bias=ws.to(BF16)), TypeError),
                       (lambda: ctx.i8_linear(x, wq, ws, residual=dy.float()), TypeError), (lambda: ctx.i8_linear(x, wq, ws, residual=dy[:5]), ValueError),
                       (lambda: ctx.i8_linear(x, wq, ws, out_dtype=torch.int8), TypeError), (lambda: ctx.i8_linear(x, wq, ws[::2].repeat(2)[::1], bias=torch.randn(16, device="cuda")[::2]), ValueError),
                       (lambda: ctx.i8_linear_grad(dy, q[:5], s[:5], wq, ws), ValueError), (lambda: ctx.i8_linear_grad(dy[:, :7], q, s, wq, ws), ValueError),
                       (lambda: ctx.i8_linear_grad(dy, q, s, wq, ws, mask=torch.zeros(6, 2, dtype=torch.uint8, device="cuda")), ValueError),
                       (lambda: ctx.i8_linear_grad(dy.sum().expand(6, 8), q, s, wq, ws), ValueError), (lambda: ctx.i8_linear_grad(dy, q, s, wq, ws, w_dtype=torch.float64), TypeError)]:
        with pytest.raises(kind):
            call()


# ---- shapes at which a call takes another way: few output channels, few rows, long and short runs ------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m,n,k", [(300, 64, 300), (5000, 39, 700), (200, 1, 500), (65, 17, 5000), (129, 65, 300), (300, 300, 115)])
def test_linear_of_few_channels_with_residual(ctx, m, n, k, dtype):
    x = some_rows(m, k, dtype, m + n)
    wq, ws = eight(n, k, m)
    wide = torch.randn(m, n + 3, generator=gen(21), device="cuda").to(dtype)
    want, t = linear_ref(*codes(x), wq, ws)
    for res in (wide[:, 1:n + 1], wide[:1, :n].expand(m, n), wide[:, 3:].contiguous()):
        y, saved = ctx.i8_linear(x, wq, ws, residual=res, relu=True, save=True)
        r = res.double().cpu()
        within(y, (want + r).clamp(min=0), t + r.abs(), dtype, 6 * 2.0 ** -24)
        on = bits(saved.mask, n)
        assert on[y.cpu() > 0].all() and not on[want + r < -8 * 2.0 ** -24 * (t + r.abs())].any()


@pytest.mark.parametrize("dtype,w_dtype,relu", [(F32, F32, True), (F16, F16, False), (BF16, F32, True), (F32, F16, False)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 4), (16, 1, 3), (7, 2100, 70), (16, 5000, 130), (3, 2049, 4), (12, 300, 1000), (16, 64, 64), (2, 1, 4100), (9, 1024, 1),
                                   (17, 65, 66), (500, 40, 1024), (40, 256, 1000), (300, 600, 64), (300, 600, 33), (20000, 300, 130), (3000, 640, 200)])
def test_grad_of_few_rows_and_few_channels(ctx, m, n, k, dtype, w_dtype, relu):
    case = grad_case(m, n, k, dtype, m + n + k, relu)
    got = ctx.i8_linear_grad(*case[:5], mask=case[5], w_dtype=w_dtype)
    check_grad(got, grad_ref(*case), m, n, dtype, w_dtype)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        part = ctx.i8_linear_grad(*case[:5], mask=case[5], w_dtype=w_dtype, need_dx=need[0], need_dw=need[1], need_db=need[2])
        assert all((p is not None) == want and (p is None or torch.equal(p, full)) for want, p, full in zip(need, part, got))


@pytest.mark.parametrize("n,k", [(70, 40), (2500, 67), (9, 3)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_grad_of_few_rows_that_are_not_finite(ctx, n, k, dtype):
    dy, q, s, wq, ws, mask = grad_case(8, n, k, dtype, 17, True)
    keep = bits(mask, n)
    keep[2], keep[3], keep[5] = False, True, False
    mask = torch.from_numpy(np.packbits(keep.numpy(), axis=1, bitorder="little")).cuda()
    ref = grad_ref(dy, q, s, wq, ws, mask)
    clean = ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask)
    check_grad(clean, ref, 8, n, dtype, dtype)
    dy = dy.clone()
    dy[2], dy[5, ::2], dy[5, 1::2] = float("nan"), float("inf"), float("-inf")             # all masked
    for a, b in zip(ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask), clean):
        assert torch.equal(a, b)
    dy[3, 7] = float("nan")                                # kept
    dx, dw, db = ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask)
    assert dx[3].isnan().all() and dw[7].isnan().all() and db[7].isnan()
    rows_, cols = [r for r in range(8) if r != 3], [c for c in range(n) if c != 7]
    assert torch.equal(dx[rows_], clean[0][rows_]) and torch.equal(dw[cols], clean[1][cols]) and torch.equal(db[cols], clean[2][cols])


def test_grad_of_few_rows_reads_strided_tensors(ctx):
    m, n, k = 11, 1100, 70
    dy, q, s, wq, ws, mask = grad_case(m, n, k, BF16, 5, True)
    ref = grad_ref(dy, q, s, wq, ws, mask)
    wide = torch.zeros(m, n + 9, dtype=BF16, device="cuda")
    wide[:, 3:3 + n] = dy
    qo = torch.zeros(m * (k + 1) + 1, dtype=torch.int8, device="cuda")[1:].view(m, k + 1)[:, :k]
    qo.copy_(q)
    wo = torch.zeros(n * k + 5, dtype=torch.int8, device="cuda")[5:].view(n, k)             # its last row ends where its memory ends
    wo.copy_(wq)
    mw = torch.zeros(m, (n + 7) // 8 + 2, dtype=torch.uint8, device="cuda")
    mw[:, 1:-1] = mask
    check_grad(ctx.i8_linear_grad(wide[:, 3:3 + n], qo, s, wo, ws, mask=mw[:, 1:-1]), ref, m, n, BF16, BF16)
    one = ctx.i8_linear_grad(dy[:1].expand(m, n), q, s, wq, ws)
    check_grad(one, grad_ref(dy[:1].expand(m, n), q, s, wq, ws, None), m, n, BF16, BF16)


# ---- the layer that is trained ------------------------------------------------------------------------------------------------------------------------------
def plain_layer(layer, x, residual=None):
    """the layer in 64 bits over the numbers that its 8-bit rows stand for, as leaves: (y, x, w, b, residual)"""
    leaf = lambda t: t.detach().double().cpu().requires_grad_()  # noqa: E731
    q, s = codes(x.reshape(-1, x.shape[-1]))
    xh = leaf((torch.from_numpy(q).double() * torch.from_numpy(s).double()[:, None]).view(x.shape))
    wq, ws = codes(layer.weight)
    wh = leaf(torch.from_numpy(wq).double() * torch.from_numpy(ws).double()[:, None])
    b = None if layer.bias is None else leaf(layer.bias)
    r = None if residual is None else leaf(residual)
    y = xh @ wh.t()
    for t in (b, r):
        y = y if t is None else y + t
    return (y.clamp(min=0) if layer.relu else y), xh, wh, b, r


@pytest.mark.parametrize("dtype,p_dtype,relu,bias", [(F32, F32, True, True), (BF16, F32, True, True), (F16, F16, False, True), (BF16, BF16, False, False)])
@pytest.mark.parametrize("shape,n", [((3, 5, 40), 24), ((1, 64), 300), ((700, 256), 256), ((130, 520), 65), ((0, 40), 24)])
def test_layer_gradients(ctx, shape, n, dtype, p_dtype, relu, bias):
    from dnascent_amd import dense8
    torch.manual_seed(5)
    layer = dense8.Dense(ctx, shape[-1], n, bias=bias, relu=relu, dtype=p_dtype)
    if bias:
        with torch.no_grad():
            layer.bias.normal_()
    m = math.prod(shape[:-1])
    x = torch.randn(shape, generator=gen(1), device="cuda").to(dtype).requires_grad_()
    res = torch.randn(shape[:-1] + (n,), generator=gen(2), device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(shape[:-1] + (n,), generator=gen(3), device="cuda").to(dtype)
    y = layer(x, res)
    y.backward(dy)
    want, xh, wh, b, r = plain_layer(layer, x, res)
    live = (y.detach().cpu() > 0) if relu else torch.ones(y.shape, dtype=torch.bool)       # a sum within a rounding of zero may fall on either side
    dz = torch.where(live, dy.cpu().double(), torch.zeros((), dtype=torch.float64)).view(m, n)
    x2, w2 = xh.detach().view(m, shape[-1]), wh.detach()
    mag = x2.abs() @ w2.abs().t() + (b.detach().abs() if bias else 0) + r.detach().abs().view(m, n)
    within(y.detach().view(m, n), want.detach().view(m, n), mag, dtype, 6 * 2.0 ** -24)
    ref = (dz @ w2, dz.t() @ x2, dz.sum(0)), (dz.abs() @ w2.abs(), dz.abs().t() @ x2.abs(), dz.abs().sum(0))
    got = (x.grad.view(m, shape[-1]), layer.weight.grad, layer.bias.grad if bias else ref[0][2].to(p_dtype).cuda())
    assert layer.weight.grad.dtype == p_dtype and x.grad.dtype == dtype
    check_grad(got, ref, m, n, dtype, p_dtype)
    assert torch.equal(res.grad.double().cpu().view(m, n), dz)
    if not relu and m:                                     # and against differences of the plain layer: linear, so a step of any size will do
        (want * dy.cpu().double()).sum().backward()
        d = torch.randn(w2.shape, dtype=torch.float64)
        up, down = ((x2 @ (w2 + f * d).t() * dz).sum() for f in (0.5, -0.5))
        assert abs((wh.grad * d).sum() - (up - down)) <= 1e-9 * (ref[1][1] * d.abs()).sum()


def test_layer_shared_broadcast_frozen_and_summed(ctx):
    from dnascent_amd import dense8
    torch.manual_seed(6)
    layer = dense8.Dense(ctx, 48, 48, relu=False)
    x = torch.randn(1, 48, device="cuda").requires_grad_()
    layer(x.expand(20, 48)).sum().backward()               # one row read twenty times; the gradient of a sum is one number repeated
    w, wx = layer.weight.grad.clone(), x.grad.clone()
    y, xh, wh, b, _ = plain_layer(layer, x)
    (20 * y.sum()).backward()
    mag = 20 * wh.detach().abs().sum(0, keepdim=True)
    within(wx, xh.grad, mag, F32, 2.0 ** -21 + 68 * 2.0 ** -24)
    within(w, wh.grad, 20 * xh.detach().abs().expand(48, 48), F32, 2.0 ** -21 + 20 * 2.0 ** -24)
    layer.zero_grad()
    a = layer(x.detach())                                  # twice through one weight: its gradients add up
    layer(a).backward(torch.ones(1, 48, device="cuda"))
    first = [p.grad.clone() for p in layer.parameters()]
    layer.zero_grad()
    mid = a.detach().requires_grad_()
    layer(mid).backward(torch.ones(1, 48, device="cuda"))
    layer(x.detach()).backward(mid.grad)
    assert all(torch.allclose(p.grad, f, rtol=2.0 ** -22, atol=1e-6) for p, f in zip(layer.parameters(), first))
    layer.zero_grad()
    layer.weight.requires_grad_(False)
    layer(x).sum().backward()
    assert layer.weight.grad is None and layer.bias.grad is not None
    with torch.no_grad():
        assert not layer(x).requires_grad
    t = torch.randn(48, 30, device="cuda").t()             # elements of a row not next to each other
    assert torch.equal(layer(t), layer(t.contiguous()))
    y = layer(x)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)                    # no second derivatives


def test_layer_run_and_captured(ctx):
    """two layers one after the other, fitted for a few steps: eagerly, and the same steps as one captured graph that is replayed with eager work in between"""
    from dnascent_amd import dense8

    def fresh():
        torch.manual_seed(7)
        return torch.nn.ModuleList([dense8.Dense(ctx, 64, 256, relu=True), dense8.Dense(ctx, 256, 64)])
    x = torch.randn(500, 64, generator=gen(1), device="cuda")
    target = torch.randn(500, 64, generator=gen(2), device="cuda")

    def step(net):
        y = net[1](net[0](x), x)
        grads = torch.autograd.grad(y, list(net.parameters()), (y.detach() - target) * (2.0 / 500))        # of the squared error's sum over channels, mean over rows
        with torch.no_grad():
            for p, g in zip(net.parameters(), grads):
                p.sub_(g, alpha=0.01)
        return y.detach()
    eager, captured = fresh(), fresh()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(fresh())
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    for rep in range(4):
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
        assert all(torch.equal(a, b) for a, b in zip(eager.parameters(), captured.parameters())), rep


def test_layer_of_a_description(ctx):
    """a pointwise convolution leaves a description, is used and fitted as a layer, and goes back: the network runs with it"""
    from dnascent_amd import cnn_model, dense8
    desc, blob, _ = cnn_model.default_model(3)
    i = next(j for j, op in enumerate(desc["ops"]) if op["op"] == "conv" and op["k"] == 1 and op["relu"])
    op = desc["ops"][i]
    layer = dense8.Dense.from_op(ctx, desc, blob, i)
    assert layer.relu and tuple(layer.weight.shape) == (op["cout"], op["cin"])
    lens = np.array([200, 90], np.uint32)
    rng = np.random.default_rng(1)
    inputs = lens, rng.integers(1, 1025, 290).astype(np.float32), rng.integers(1, 257, 290).astype(np.float32), rng.normal(0, 1, (290, 20)).astype(np.float32)

    def probabilities(b):
        c = hip.Context(0)
        c.load_cnn(desc, b)
        p = c.cnn_infer(*inputs)
        c.close()
        return p
    same, moved = blob.copy(), blob.copy()
    layer.store(desc, same, i)
    k, n = op["cin"], op["cout"]
    folded = blob[op["w"]:op["w"] + k * n].reshape(k, n) * blob[op["scale"]:op["scale"] + n]
    assert np.array_equal(same[op["w"]:op["w"] + k * n].reshape(k, n), folded) and (same[op["scale"]:op["scale"] + n] == 1).all()
    before = probabilities(blob)
    assert np.abs(probabilities(same) - before).max() < 1e-4               # the factor is in the kernel now: roundings only
    x = torch.randn(290, k, generator=gen(4), device="cuda")
    layer(x).square().sum(-1).mean().backward()
    with torch.no_grad():
        for p in layer.parameters():
            p.sub_(p.grad, alpha=0.5)
    layer.store(desc, moved, i)
    assert np.array_equal(moved[op["w"]:op["w"] + k * n].reshape(k, n), layer.weight.detach().cpu().numpy().T)
    after = probabilities(moved)
    assert np.abs(after - before).max() > 1e-4 and np.allclose(after.sum(1), 1, atol=1e-5)
    back = dense8.Dense.from_op(ctx, desc, moved, i)
    assert torch.equal(back.weight, layer.weight) and torch.equal(back.bias, layer.bias)


def test_layer_refusals(ctx):
    from dnascent_amd import cnn_model, dense8
    desc, blob, _ = cnn_model.default_model(3)
    layer = dense8.Dense(ctx, 8, 4)
    with pytest.raises(ValueError):
        layer(torch.zeros(3, 9, device="cuda"))
    with pytest.raises(ValueError):
        layer(torch.zeros(3, 8))
    with pytest.raises(ValueError):
        layer(torch.zeros(3, 8, device="cuda", dtype=torch.int8))
    with pytest.raises(TypeError):
        dense8.Dense(ctx, 8, 4, dtype=torch.float64)
    with pytest.raises(ValueError):
        dense8.Dense.from_op(ctx, desc, blob, 0)
    i = next(j for j, op in enumerate(desc["ops"]) if op["op"] == "conv" and op["k"] == 1)
    with pytest.raises(ValueError):
        layer.store(desc, blob, i)


def test_more_rows_than_one_launch_has(ctx):
    m, k = 2 ** 23 + 5, 3
    x = torch.randn(m, k, generator=gen(51), device="cuda").to(BF16)
    q, s = ctx.i8_rows(x)
    y = ctx.i8_restore(q, s, BF16)
    for part in (slice(0, 3), slice(2 ** 23 - 3, m)):
        qr, sr = codes(x[part])
        assert np.array_equal(q[part].cpu().numpy(), qr) and s[part].cpu().numpy().tobytes() == sr.tobytes()
        want = torch.from_numpy(qr).double() * torch.from_numpy(sr).double()[:, None]
        within(y[part], want, want.abs(), BF16, 2.0 ** -24)
    n = 257                                                # dx of a wide layer: rows of dz sw first
    wq, ws = eight(n, k, 52)
    dy = torch.zeros(m, n, dtype=BF16, device="cuda")
    at = torch.tensor([0, 1, 2 ** 23 - 1, 2 ** 23, m - 1], device="cuda")
    dy[at] = torch.randn(5, n, generator=gen(53), device="cuda").to(BF16)
    dx, _, _ = ctx.i8_linear_grad(dy, q, s, wq, ws, need_dw=False, need_db=False)
    (want, _, _), (t, _, _) = grad_ref(dy[at], q[at], s[at], wq, ws, None)
    within(dx[at], want, t, BF16, 2.0 ** -11 + n * 2.0 ** -24)
    assert int((dx != 0).any(1).sum()) == 5


def test_layer_copied_one_row_and_state(ctx):
    import copy

    from dnascent_amd import dense8
    layer = dense8.Dense(ctx, 40, 24, relu=True)
    twin = copy.deepcopy(torch.nn.Sequential(layer))[0]
    assert twin.ctx is ctx and torch.equal(twin.weight, layer.weight) and twin.weight.data_ptr() != layer.weight.data_ptr()
    x = torch.randn(40, device="cuda").requires_grad_()    # no leading dimension at all
    res = torch.randn(24, device="cuda").requires_grad_()
    y = layer(x, res)
    assert y.shape == (24,) and torch.equal(y, layer(x[None], res[None])[0])
    y.sum().backward()
    assert x.grad.shape == (40,) and torch.equal(res.grad, (y > 0).float())
    with torch.no_grad():
        twin.weight.zero_()
    twin.load_state_dict(layer.state_dict())
    assert torch.equal(twin(x, res), y)
    other = layer(x)                                       # the weight may change between the passes: what was multiplied is what is differentiated
    want, = torch.autograd.grad(layer(x).sum(), x)
    with torch.no_grad():
        layer.weight.mul_(3)
    got, = torch.autograd.grad(other.sum(), x)
    assert torch.equal(got, want)


def test_calls_and_refusals_from_several_threads(ctx):
    """one context, four threads with a stream each: results as alone, and errors that overlap are errors and nothing worse"""
    import threading
    calls = [_mixed(ctx, 900, 256, 256, BF16, 61), _mixed(ctx, 12, 520, 384, F16, 62), _mixed(ctx, 300, 64, 64, F32, 63), _mixed(ctx, 70, 130, 700, BF16, 64)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    bad = []
    d = hip.i8_desc(hip.I8_LINEAR_FIELDS, m=3, n=-5, k=7)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = calls[i]()
                    need = C.c_uint64(0)
                    if hip.lib().dn_i8_linear_workspace(ctx.h, d, C.byref(need)) == 0 or not hip.lib().dn_last_error(ctx.h):
                        bad.append(("not refused", i))
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(("differs", i))
        except Exception as e:  # noqa: BLE001
            bad.append((repr(e), i))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:4]


# ---- results whose own terms are small beside their row's or channel's ------------------------------------------------------------------------------------
def _outliers(m, n, k, dtype, far, seed):
    """a few rows of dy are 2^far above the others and a few channels 2^far above those beside them; the codes that stand under them (q's for dw, wq's for dx) are
    zero in every second column, so that half of the results have small terms only"""
    dy, q, s, wq, ws, mask = grad_case(m, n, k, F32, seed, True)
    dy = torch.randn(m, n, generator=gen(seed + 5), device="cuda") * 2.0 ** -8
    rows_, cols = [0, m // 2, m - 1], [1 % n, n // 2, n - 1]
    q[rows_, ::2] = 0
    wq[cols, ::2] = 0
    by_row, by_col = dy.clone(), dy.clone()
    by_row[rows_] *= 2.0 ** far
    by_col[:, cols] *= 2.0 ** far
    return by_row.to(dtype), by_col.to(dtype), q, s, wq, ws, mask


@pytest.mark.parametrize("dtype,w_dtype,far", [(F32, F32, 20), (F32, F32, 36), (F32, F32, 70), (BF16, BF16, 30), (BF16, F32, 60), (F16, F16, 20), (F32, F16, 40)])
@pytest.mark.parametrize("m,n,k", [(12, 700, 90), (16, 64, 2000), (300, 64, 64), (65, 40, 3), (500, 100, 130), (3000, 256, 256), (40000, 250, 200), (33, 1000, 40), (600, 300, 520),
                                   (900, 5000, 2), (100, 9000, 70), (70, 1500, 300)])
def test_grad_of_results_with_small_terms_only(ctx, m, n, k, dtype, w_dtype, far):
    by_row, by_col, q, s, wq, ws, mask = _outliers(m, n, k, dtype, far, m + n + k)
    for dy in (by_row, by_col):
        for mk in (None, mask):
            got, ref = ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mk, w_dtype=w_dtype), grad_ref(dy, q, s, wq, ws, mk)
            piece = [2.0 ** -21 if t == F32 else 2.0 ** -11 for t in (dtype, w_dtype)]
            room = piece[0] + n * 2.0 ** -24, piece[1] + m * 2.0 ** -24, m * 2.0 ** -24               # as check_grad has them
            check_grad([_border(*v) for v in zip(got, *ref, room)], ref, m, n, dtype, w_dtype)


def _border(got, want, terms, u):
    """Infinity is the right rounding of everything from half a step above the type's largest number on (fp16's largest is 65504, the step there 32: 65520 becomes infinity),
    so a result that may lie anywhere within its room of `want` may be infinite if want plus room reaches that.  within() only asks for infinity where want minus room
    is above the largest number; in between both are right, and the largest number (which is within the room) stands in for infinity."""
    top, half = torch.finfo(got.dtype).max, HALF[got.dtype]
    want, terms = want.to(got.device), terms.to(got.device)
    room = half * want.abs() + u * terms
    near = (want.abs() - room <= top) & (want.abs() + room >= top * (1 + half)) & (got == want.sign() * math.inf)
    return torch.where(near, (want.sign() * top).to(got.dtype), got)


def test_a_workspace_of_another_description_is_refused(ctx):
    """the size for rows at multiples of 16 bytes does not do for the same shape elsewhere; the size for the call itself does"""
    L = hip.lib()
    m, n, k = 200, 300, 297
    x = some_rows(m, k, BF16, 71)
    q, s = ctx.i8_rows(x)
    wq, ws = eight(n, k, 72)
    odd = torch.zeros(n * k + 1, dtype=torch.int8, device="cuda")[1:].view(n, k)
    odd.copy_(wq)
    y = torch.empty(m, n, dtype=BF16, device="cuda")

    def desc(w):
        return hip.i8_desc(hip.I8_LINEAR_FIELDS, m=m, n=n, k=k, x=q.data_ptr(), ldx=q.stride(0), sx=s.data_ptr(), w=w.data_ptr(), ldw=w.stride(0), sw=ws.data_ptr(),
                           y=y.data_ptr(), ldy=n, x_type=3, y_type=2)
    need = [C.c_uint64(0), C.c_uint64(0)]
    for w, v in zip((wq, odd), need):
        assert L.dn_i8_linear_workspace(ctx.h, desc(w), C.byref(v)) == 0
    assert need[1].value > need[0].value
    space = torch.empty(need[1].value, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    assert L.dn_i8_linear(ctx.h, desc(odd), space.data_ptr(), need[0].value, st) == -3 and b"workspace" in L.dn_last_error(ctx.h)
    assert L.dn_i8_linear(ctx.h, desc(odd), space.data_ptr(), need[1].value, st) == 0
    assert torch.equal(y, ctx.i8_linear(q, wq, ws, sx=s))


def test_calls_without_a_history(ctx):
    """a tensor that requires a gradient: refused, but taken under no_grad and detached; i8_rows makes a parameter's rows"""
    wq, ws = eight(24, 40, 81)
    x = some_rows(30, 40, BF16, 82).requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        ctx.i8_linear(x, wq, ws)
    y = ctx.i8_linear(x.detach(), wq, ws)
    with torch.no_grad():
        assert torch.equal(ctx.i8_linear(x, wq, ws), y)
    q, s = ctx.i8_rows(x)
    assert not s.requires_grad and torch.equal(q, ctx.i8_rows(x.detach())[0])


@pytest.mark.parametrize("m,n,k", [(3, 24, 40), (700, 256, 256), (2000, 300, 520)])
def test_layer_without_gradients_keeps_nothing(ctx, m, n, k, monkeypatch):
    from dnascent_amd import dense8
    layer = dense8.Dense(ctx, k, n, relu=True)
    x, res = some_rows(m, k, BF16, 91), some_rows(m, n, BF16, 92)
    want = layer(x, res)
    assert want.requires_grad
    kept = []
    plain = dense8.linear
    monkeypatch.setattr(dense8, "linear", lambda *a, **kw: kept.append(kw.get("save", False)) or plain(*a, **kw))
    with torch.no_grad():
        y = layer(x.clone().requires_grad_(), res)
    assert torch.equal(y, want.detach()) and not y.requires_grad
    for p in layer.parameters():
        p.requires_grad_(False)
    y = layer(x, res)                                      # gradients are on, and nothing asks for one
    assert torch.equal(y, want.detach()) and not y.requires_grad
    assert kept == [False, False]
    layer.bias.requires_grad_(True)
    assert layer(x, res).requires_grad and kept[-1]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,n,k", [(9, 60, 40), (16, 300, 90), (200, 64, 64), (300, 128, 100), (20000, 250, 70), (400, 700, 130)])
def test_grad_with_channel_scales_far_apart_and_zero(ctx, m, n, k, relu, dtype):
    """output channels whose weights are 2^-30 to 2^6 of each other, some of them nothing at all (a dead channel), and a layer of dead channels only"""
    dy, q, s, wq, ws, mask = grad_case(m, n, k, dtype, 7 * m + n, relu)
    ws = ws * torch.exp2(torch.randint(-30, 7, (n,), generator=gen(n), device="cuda").float())
    ws[::5] = 0
    ws[n // 2] = 2.0 ** 10
    got, ref = ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask), grad_ref(dy, q, s, wq, ws, mask)
    check_grad(got, ref, m, n, dtype, dtype)
    dead = torch.zeros_like(ws)
    dx, dw, db = ctx.i8_linear_grad(dy, q, s, wq, dead, mask=mask)
    assert not dx.any() and torch.equal(dw, got[1]) and torch.equal(db, got[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [-75, 60])
@pytest.mark.parametrize("m,n,k", [(300, 64, 64), (3000, 256, 256), (600, 300, 520)])
def test_grad_of_small_terms_near_the_ends_of_the_range(ctx, m, n, k, shift, dtype):
    """the same, with every number 2^-75 or 2^60 of what it was: factors down to 2^-100, and large ones far from fp32's end still"""
    by_row, by_col, q, s, wq, ws, mask = _outliers(m, n, k, F32, 34, m + n)
    for dy in (by_row, by_col):
        dy = (dy * 2.0 ** shift).to(dtype)
        check_grad(ctx.i8_linear_grad(dy, q, s, wq, ws, mask=mask), grad_ref(dy, q, s, wq, ws, mask), m, n, dtype, dtype)
