"""The 8-bit dense layer of dnascent_amd, measured: cases, inputs, the plain forms and what a pass has to move.

Three operators, M rows (positions of reads, or tokens), K input channels, N output channels:

  checkpoint   rows of x are stored as 8-bit integers with one scale each, and restored
               a = max_k |x|, q = rint(x * (127 / a)), s = a / 127 (each operation in fp32), restored value q * s
  linear       y = act(s[m] * ws[n] * sum_k q[m, k] wq[n, k] + bias[n] + residual[m, n]); x comes as numbers, or as (q, s) already
  grad         of linear, from the 8-bit checkpoint of its input and, behind a ReLU, one bit per output:
               dz = dy where the bit is set; dx = (dz * ws) wq, dw = dz^T (q * s), db = sum_m dz
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST_BYTES, MOST_FLOPS = 2.5e9, 5.6e11                     # no drawn case moves or computes more than the largest listed ones


def listed():
    return [
        # one position through a layer of the detect network's last stage: a call's latency
        dict(name="linear one row", op="linear", m=1, n=256, k=256, type="bf16", relu=False, residual=False, given=False),
        # one token through a wide layer: the weights are read once, for one row
        dict(name="linear one row wide", op="linear", m=1, n=4096, k=4096, type="bf16", relu=False, residual=False, given=False),
        # a few rows whose 8-bit form the caller has already, over the 17 x 256 inputs of the network's widest window, an odd number of outputs
        dict(name="linear few rows", op="linear", m=13, n=1000, k=4352, type="f16", relu=True, residual=True, given=True),
        # a quarter of one pass of the network's rows through a 256-channel pointwise layer, in the network's own type
        dict(name="linear network pass", op="linear", m=1 << 20, n=256, k=256, type="f32", relu=True, residual=False, given=False),
        # a wide layer over a batch: the product itself
        dict(name="linear wide", op="linear", m=8192, n=4096, k=4096, type="bf16", relu=False, residual=False, given=False),
        # the gradient over one short read, 64 channels: a call's latency
        dict(name="grad short read", op="grad", m=200, n=64, k=64, type="f32", relu=True),
        # one 50 kb read, widths that no tile divides
        dict(name="grad odd widths", op="grad", m=46993, n=131, k=77, type="f16", relu=False),
        # a training batch through a 256-channel pointwise layer
        dict(name="grad network batch", op="grad", m=1 << 20, n=256, k=256, type="bf16", relu=True),
        # the gradient of the wide layer
        dict(name="grad wide", op="grad", m=8192, n=4096, k=4096, type="bf16", relu=False),
        # one row of the network's narrowest layer
        dict(name="checkpoint one row", op="checkpoint", m=1, k=64, type="f32"),
        # one long read's windows, an odd row length
        dict(name="checkpoint odd rows", op="checkpoint", m=5001, k=4353, type="f16"),
        # half of one pass of the network's rows, 256 channels
        dict(name="checkpoint network pass", op="checkpoint", m=1 << 21, k=256, type="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; every second one as it falls, the others a multiple of 32 or 64 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v -= v % (64 if v >= 512 else 32)
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(("linear", "linear", "grad", "grad", "checkpoint"))
    kind = rng.choice(sorted(TYPES))
    while True:
        m = _log(rng, 1, 1 << 20) if rng.random() < 0.8 else rng.randint(1, 16)
        n, k = _log(rng, 16, 4096), _log(rng, 16, 4352)
        case = dict(op=op, m=m, k=k, type=kind)
        if op != "checkpoint":
            case.update(n=n, relu=rng.random() < 0.5)
        if op == "linear":
            case.update(residual=rng.random() < 0.3, given=rng.random() < 0.3)
        w = work(case)
        # the plain form keeps a handful of fp32 copies of what it reads and writes
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


def _pitched(q):
    """8-bit rows as the checkpoint lays them out: each row starts at a multiple of 16 bytes, zeros behind its end."""
    m, k = q.shape
    full = torch.zeros(m, -(-k // 16) * 16, dtype=torch.int8, device=q.device)
    full[:, :k] = q
    return full[:, :k]


def _some_activations(case, g):
    """What stands before a dense layer: values around zero, channels of different sizes; behind a ReLU half of them are zero."""
    x = torch.randn(case["m"], case["k"], generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(case["k"], generator=g, device="cuda"))
    return x.clamp_(min=0) if case.get("relu") else x


def _eight_bits(x):
    a = x.abs().amax(1, keepdim=True)
    return torch.round(x * (127.0 / a.clamp(min=1e-30))).to(torch.int8), (a / 127.0).squeeze(1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["type"]]
    m, k = case["m"], case["k"]
    state = dict(case=case)
    x = _some_activations(case, g)
    if case["op"] == "checkpoint":
        state["x"] = x.to(t)
        return state
    n = case["n"]
    wq, state["ws"] = _eight_bits(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
    state["wq"] = _pitched(wq)
    if case["op"] == "linear":
        if case["given"]:
            q, state["sx"] = _eight_bits(x)
            state["x"] = _pitched(q)
        else:
            state["x"] = x.to(t)
        state["bias"] = 0.1 * torch.randn(n, generator=g, device="cuda")
        state["residual"] = torch.randn(m, n, generator=g, device="cuda").to(t) if case["residual"] else None
        return state
    q, state["s"] = _eight_bits(x)
    state["q"] = _pitched(q)
    # gradients of a mean over positions: small, and not of one size in every row
    dy = torch.randn(m, n, generator=g, device="cuda")
    dy *= 1e-3 * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    state["dy"] = dy.to(t)
    state["mask"] = torch.randint(0, 256, (m, -(-n // 8)), generator=g, device="cuda", dtype=torch.uint8) if case["relu"] else None
    return state


_contexts = {}


def _context():
    from dnascent_amd import hip
    d = torch.cuda.current_device()
    if d not in _contexts:
        _contexts[d] = hip.Context(d)
    return _contexts[d]


def _plain_rows(x):
    """The 8-bit rows of x and their scales, both as fp32 numbers.  (Tensors on both sides of a division: torch multiplies by a rounded
    reciprocal where one side is a Python number, and a code next to a border then falls on the other side.)"""
    x = x.float()
    a = x.abs().amax(1, keepdim=True)
    top = torch.full_like(a, 127.0)
    r = torch.where(a >= 2.0 ** -120, top / a, torch.zeros_like(a))
    return torch.round(x * r), torch.where(a >= 2.0 ** -120, a / top, torch.zeros_like(a))


def _plain_bits(mask, n):
    bits = torch.arange(8, device=mask.device, dtype=torch.uint8)
    return ((mask.unsqueeze(2) >> bits) & 1).reshape(mask.shape[0], -1)[:, :n].bool()


def run(state):
    case = state["case"]
    t = TYPES[case["type"]]
    if case["op"] == "checkpoint":
        if own:
            ctx = _context()
            q, s = ctx.i8_rows(state["x"])
            return dict(x=ctx.i8_restore(q, s, t), s=s)
        q, s = _plain_rows(state["x"])
        return dict(x=(q * s).to(t), s=s.squeeze(1))
    if case["op"] == "linear":
        if own:
            return _context().i8_linear(state["x"], state["wq"], state["ws"], sx=state.get("sx"), bias=state["bias"],
                                        residual=state["residual"], relu=case["relu"], out_dtype=t)
        if case["given"]:
            x = state["x"].float() * state["sx"].unsqueeze(1)
        else:
            q, s = _plain_rows(state["x"])
            x = q * s
        y = x @ (state["wq"].float() * state["ws"].unsqueeze(1)).t() + state["bias"]
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return (torch.clamp(y, min=0) if case["relu"] else y).to(t)
    if own:
        dx, dw, db = _context().i8_linear_grad(state["dy"], state["q"], state["s"], state["wq"], state["ws"], mask=state["mask"])
        return dict(dx=dx, dw=dw, db=db)
    dz = state["dy"].float()
    if state["mask"] is not None:
        dz = torch.where(_plain_bits(state["mask"], case["n"]), dz, torch.zeros_like(dz))
    dx = dz @ (state["wq"].float() * state["ws"].unsqueeze(1))
    dw = dz.t() @ (state["q"].float() * state["s"].unsqueeze(1))
    return dict(dx=dx.to(t), dw=dw.to(t), db=dz.sum(0).to(t))


def work(case):
    m, k, e = case["m"], case["k"], BYTES[case["type"]]
    if case["op"] == "checkpoint":                         # x in, 8 bits out; 8 bits in, x out
        return dict(bytes=2 * (m * k * e + m * k + 4 * m), flops=4 * m * k)
    n = case["n"]
    if case["op"] == "linear":
        x = m * (k + 4) if case["given"] else m * k * e
        return dict(bytes=x + n * k + 8 * n + m * n * e * (2 if case["residual"] else 1), flops=2 * m * n * k)
    mask = m * (-(-n // 8)) if case["relu"] else 0
    return dict(bytes=m * n * e + mask + m * (k + 4) + n * (k + 4) + m * k * e + n * k * e + n * e, flops=4 * m * n * k)


def exact(case, seed):
    """From the definition, in 64 bits.  Which 8-bit number a value becomes is part of the definition (fp32 operations, in this order);
    everything after that -- products, sums, scales -- is done here in 64 bits, the sums over integers without any rounding of the operands."""
    state = prepare(case, seed)

    def codes(x):
        x = x.to(torch.float32)
        top = torch.maximum(x.amax(1), -x.amin(1))
        live = top >= 2.0 ** -120
        mult = torch.zeros_like(top)
        mult[live] = torch.full_like(top[live], 127.0) / top[live]
        scale = torch.zeros_like(top)
        scale[live] = top[live] / torch.full_like(top[live], 127.0)
        return (x * mult[:, None]).round_().double(), scale

    if case["op"] == "checkpoint":
        q, s = codes(state["x"])
        q *= s.double()[:, None]
        return dict(x=q, s=s.double())
    wq, ws = state["wq"].double(), state["ws"].double()
    if case["op"] == "linear":
        q, s = (state["x"].double(), state["sx"]) if case["given"] else codes(state["x"])
        y = torch.mm(q, wq.t().contiguous())               # whole numbers below 2^53: no rounding
        y *= s.double()[:, None]
        y *= ws[None, :]
        y += state["bias"].double()[None, :]
        if state["residual"] is not None:
            y += state["residual"].double()
        return y.clamp_(min=0.0) if case["relu"] else y
    dz = state["dy"].double()
    if state["mask"] is not None:
        n = torch.arange(case["n"], device=dz.device)
        keep = (state["mask"][:, n // 8].int() >> (n % 8).int()) % 2 == 1
        dz.masked_fill_(~keep, 0.0)
    db = dz.sum(0)
    dx = torch.mm(dz * ws[None, :], wq)
    dz *= state["s"].double()[:, None]
    return dict(dx=dx, dw=torch.mm(dz.t().contiguous(), state["q"].double()), db=db)
