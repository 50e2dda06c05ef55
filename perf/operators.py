"""Cases of the training operators around the fused MLP: what is measured, and their plain forms.

Three operators, each of which a training step of the MLP block calls next to the MLP's own forward and backward pass:

  norm     layer norm and RMS norm of the rows of a matrix, forward and backward; the backward pass also reduces the
           gradients of the weight and the bias over the rows, and adds the gradient that reaches the input past the norm
  adamw    one AdamW step over many tensors at once, with the two moments in 32 bits or in 8
  clip     the 2-norm over many gradients at once, and the factor that clips it

8-bit moments.  A tensor's moments are cut into blocks of 256 elements (the last may be shorter), and each block has a
power of two as its scale: the first moment is float8_e4m3fn times its scale, whose largest magnitude lies in [2^7, 2^8)
before rounding, the second is float8_e5m2 times its scale, whose largest lies in [2^14, 2^15).  Both are rounded
stochastically, with 16 random bits for each value that are a function of the seed, the step and the value's position, so
that the averages do not stall where a step changes them by less than half a unit; a second moment above zero is never
rounded to zero.  A position counts whole blocks: the tensors of a call take their blocks one after the other.
"""
import math
import sys

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.1, 100
BLOCK = 256
# odd multipliers: value i of a group of eight takes its 32 random bits from hash * MULT[i]
MULT = (0x5ECD29B7, 0xDB623B29, 0x69758763, 0x7D45CE1D, 0x74A1B41D, 0x75BBB081, 0x5AD24435, 0x73B07CC5)
M32 = 0xFFFFFFFF
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one serving batch of sixteen tokens through a norm of width 4096: latency
        {"name": "layer_fwd_16x4096", "op": "norm", "pass": "fwd", "kind": "layer", "rows": 16, "cols": 4096,
         "type": "bf16", "wtype": "bf16", "bias": True, "res": False},
        # the 7B prefill batch
        {"name": "layer_fwd_4096x4096", "op": "norm", "pass": "fwd", "kind": "layer", "rows": 4096, "cols": 4096,
         "type": "bf16", "wtype": "bf16", "bias": True, "res": False},
        # the ragged 13B batch, the norm of Llama-family blocks
        {"name": "rms_fwd_32414x5120", "op": "norm", "pass": "fwd", "kind": "rms", "rows": 32414, "cols": 5120,
         "type": "bf16", "wtype": "bf16", "bias": False, "res": False},
        # an odd width in 32 bits: rows that start on no vector boundary
        {"name": "layer_bwd_1000x1003_fp32", "op": "norm", "pass": "bwd", "kind": "layer", "rows": 1000, "cols": 1003,
         "type": "fp32", "wtype": "fp32", "bias": True, "res": False},
        # the 7B training batch of a pre-norm block: the residual's gradient joins here
        {"name": "layer_bwd_4096x4096", "op": "norm", "pass": "bwd", "kind": "layer", "rows": 4096, "cols": 4096,
         "type": "bf16", "wtype": "bf16", "bias": True, "res": True},
        # the ragged 13B batch
        {"name": "rms_bwd_32414x5120", "op": "norm", "pass": "bwd", "kind": "rms", "rows": 32414, "cols": 5120,
         "type": "bf16", "wtype": "bf16", "bias": False, "res": True},
        # two small odd matrices in 32 bits with 8-bit moments: latency
        {"name": "adamw8_2x570k", "op": "adamw", "tensors": 2, "size": 569921, "ragged": False, "ptype": "fp32",
         "gtype": "fp32", "master": False, "bits": 8},
        # many small tensors of uneven sizes, as adapters and norm vectors are; 32-bit copies beside bf16 weights
        {"name": "adamw32_224x65k", "op": "adamw", "tensors": 224, "size": 65536, "ragged": True, "ptype": "bf16",
         "gtype": "bf16", "master": True, "bits": 32},
        # the three matrices of a 7B MLP, moments and weights' copies in 32 bits
        {"name": "adamw32_3x11008x4096", "op": "adamw", "tensors": 3, "size": 45088768, "ragged": False, "ptype": "bf16",
         "gtype": "bf16", "master": True, "bits": 32},
        # the same with 8-bit moments
        {"name": "adamw8_3x11008x4096", "op": "adamw", "tensors": 3, "size": 45088768, "ragged": False, "ptype": "bf16",
         "gtype": "bf16", "master": True, "bits": 8},
        # the norm over the many small gradients
        {"name": "clip_224x65k", "op": "clip", "tensors": 224, "size": 65536, "ragged": True, "gtype": "bf16"},
        # the norm over the gradients of a 7B MLP, kept in 32 bits
        {"name": "clip_3x11008x4096_fp32", "op": "clip", "tensors": 3, "size": 45088768, "ragged": False, "gtype": "fp32"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("norm", "norm", "adamw", "adamw", "clip"))
    if op == "norm":
        kind = rng.choice(("layer", "rms"))
        t = rng.choice(("bf16", "bf16", "fp32"))
        cols = spread(64, 8192)
        if rng.random() < 0.6:
            cols = (cols + 7) // 8 * 8
        most = 32414 * 5120 // (cols * (2 if t == "fp32" else 1))
        side = rng.choice(("fwd", "bwd"))
        return {"op": "norm", "pass": side, "kind": kind, "rows": spread(1, min(32768, most)),
                "cols": cols, "type": t, "wtype": rng.choice((t, "fp32")), "bias": kind == "layer" and rng.random() < 0.8,
                "res": side == "bwd" and rng.random() < 0.5}
    total = spread(4096, 100_000_000)
    tensors = min(spread(1, 256), total // 64)
    case = {"op": op, "tensors": tensors, "size": max(1, total // tensors), "ragged": rng.random() < 0.5}
    if op == "clip":
        return dict(case, gtype=rng.choice(("bf16", "fp32")))
    ptype = rng.choice(("bf16", "bf16", "fp32"))
    return dict(case, ptype=ptype, gtype="fp32" if ptype == "fp32" else rng.choice(("bf16", "fp32")),
                master=ptype == "bf16" and rng.random() < 0.5, bits=rng.choice((32, 8)))


def _sizes(case):
    n, size = case["tensors"], case["size"]
    if not case["ragged"]:
        return [size] * n
    # between a quarter and seven quarters of the usual size, every third one odd
    return [max(1, size * (1 + i * 5 % 7) // 4 + (i % 3 == 1)) for i in range(n)]


def _flat(sizes):
    """Where each tensor starts in one buffer, on whole blocks, and the buffer's length."""
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return starts, at


def _views(buffer, starts, sizes):
    return [buffer[s:s + n] for s, n in zip(starts, sizes)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        t, wt = TYPES[case["type"]], TYPES[case["wtype"]]
        # activations: rows of different size, off zero, with the large values that a few channels have
        x = randn(rows, cols) * torch.exp(0.5 * randn(rows, 1)) + 0.3 * randn(rows, 1)
        x = (x * torch.where(torch.rand((1, cols), generator=g, device=dev) < 0.01, 8.0, 1.0)).to(t)
        s = {"case": case, "x": x, "w": (1 + 0.1 * randn(cols)).to(wt),
             "b": (0.1 * randn(cols)).to(wt) if case["bias"] else None}
        if case["pass"] == "bwd":
            s["dy"] = (randn(rows, cols) * 0.02).to(t)
            s["res"] = (randn(rows, cols) * 0.02).to(t) if case["res"] else None
            x64 = x.double()
            mean = x64.mean(1) if case["kind"] == "layer" else torch.zeros(rows, dtype=torch.float64, device=dev)
            s["mean"] = mean.float()
            s["rstd"] = torch.rsqrt((x64 - mean[:, None]).square().mean(1) + 1e-5).float()
        return s

    sizes = _sizes(case)
    starts, total = _flat(sizes)
    at = torch.tensor(starts, device=dev)
    inside = torch.arange(total, device=dev)
    of = torch.bucketize(inside, at, right=True) - 1
    inside = inside - at[of] < torch.tensor(sizes, device=dev)[of]
    # gradients whose size differs from row to row
    spread = torch.exp(randn(total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-3
    grad = torch.where(inside, randn(total) * spread, 0.0).to(TYPES[case["gtype"]])
    s = {"case": case, "g": grad, "grads": _views(grad, starts, sizes)}
    if case["op"] == "clip":
        return s
    p = torch.where(inside, randn(total) * 0.02, 0.0)
    m = torch.where(inside, randn(total) * spread * 0.3, 0.0)
    v = torch.where(inside, (randn(total) * 0.3 + 1).square() * spread.square(), 0.0)
    s["p"] = p.to(TYPES[case["ptype"]])
    s["master"] = s["p"].float() + torch.where(inside, randn(total) * 1e-5, 0.0) if case["master"] else None
    if case["bits"] == 8:
        for name, x, t, top in (("m", m, torch.float8_e4m3fn, 7), ("v", v, torch.float8_e5m2, 14)):
            x = x.view(-1, BLOCK)
            _, e = torch.frexp(x.abs().amax(1))
            scale = torch.ldexp(torch.ones_like(x[:, 0]), torch.clamp(e - 1 - top, min=-126))
            s[name], s[name + "s"] = (x / scale[:, None]).to(t).view(-1), scale
    else:
        s["m"], s["v"], s["ms"], s["vs"] = m, v, None, None
    blocks = [(n + BLOCK - 1) // BLOCK for n in sizes]
    for name in ("p", "m", "v", "master"):
        s[name + "_list"] = [] if s[name] is None else _views(s[name], starts, sizes)
    for name in ("ms", "vs"):
        s[name + "_list"] = [] if s[name] is None else _views(s[name], [a // BLOCK for a in starts], blocks)
    s["clip"] = torch.tensor([0.5], device=dev)
    s["seed"] = seed
    return s


def _mix32(x):
    """Two rounds of xor-shift and multiplication on 32 bits: of a number, or of a tensor that holds them in int64."""
    x = ((x ^ (x >> 16)) * 0xDDC24D79) & M32
    x = ((x ^ (x >> 15)) * 0x77D0AC3D) & M32
    return x ^ (x >> 16)


def _random_bits(total, seed, device):
    """32 bits for each of `total` positions, in int64: the upper 16 for the second moment, the lower for the first."""
    key = _mix32((seed & M32) ^ _mix32((STEP ^ (seed >> 32)) & M32))
    group = torch.arange(total // 8, device=device)
    h = _mix32((group & M32) ^ ((group >> 32) * MULT[0] & M32) ^ key)
    return ((h[:, None] * torch.tensor(MULT, device=device)) & M32).view(-1)


def _framework():
    if "fused-swiglu_b200" not in sys.path:
        sys.path.insert(0, "fused-swiglu_b200")
    import fused_mlp_module

    return fused_mlp_module


def _norm_own(s):
    c, lib = s["case"], _framework()
    if c["pass"] == "fwd":
        if c["kind"] == "layer":
            return lib.layer_norm_forward(s["x"], s["w"], s["b"], 1e-5)
        return lib.rms_norm_forward(s["x"], s["w"], 1e-5)
    if c["kind"] == "layer":
        return lib.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"], c["bias"], s["res"])
    return lib.rms_norm_backward(s["dy"], s["x"], s["rstd"], s["w"], s["res"])


def _norm_plain(s):
    c, x, w = s["case"], s["x"].float(), s["w"].float()
    if c["pass"] == "fwd":
        mean = x.mean(1) if c["kind"] == "layer" else None
        z = x - mean[:, None] if c["kind"] == "layer" else x
        rstd = torch.rsqrt((z * z).mean(1) + 1e-5)
        y = z * rstd[:, None] * w
        if s["b"] is not None:
            y = y + s["b"].float()
        y = y.to(s["x"].dtype)
        return (y, mean, rstd) if c["kind"] == "layer" else (y, rstd)
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    z = (x - s["mean"][:, None] if c["kind"] == "layer" else x) * rstd
    a = dy * w
    dx = a - z * (a * z).mean(1, keepdim=True)
    if c["kind"] == "layer":
        dx = dx - a.mean(1, keepdim=True)
    dx = dx * rstd
    if s["res"] is not None:
        dx = dx + s["res"].float()
    dx = dx.to(s["x"].dtype)
    dw = (dy * z).sum(0, dtype=torch.float64).to(s["w"].dtype)
    if c["kind"] == "rms":
        return dx, dw
    return dx, dw, dy.sum(0, dtype=torch.float64).to(s["w"].dtype) if c["bias"] else None


def _adamw_own(s):
    _framework().adamw_step(s["p_list"], s["grads"], s["m_list"], s["v_list"], STEP, LR, BETA1, BETA2, EPS, DECAY,
                            s["master_list"], s["ms_list"], s["vs_list"], s["clip"], s["seed"])
    return {k: s[k] for k in ("p", "master", "m", "v", "ms", "vs") if s[k] is not None}


def _decode(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _encode(x, bits, top, mantissa, low, least):
    """Eight-bit floats of `mantissa` bits for the blocks of x >= 0, as whole numbers, and the blocks' scales."""
    rows = x.view(-1, BLOCK)
    field = torch.clamp(rows.amax(1).view(torch.int32) >> 23, min=top + 1)
    scale = ((field - top) << 23).view(torch.float32)
    inverse = ((254 + top - field) << 23).view(torch.float32)
    # brought to where the 8-bit type's exponents, its subnormal ones too, are those of 32 bits
    y = (rows * inverse[:, None] * 2.0 ** (low - 127)).view(torch.int32).view(-1)
    drop = 23 - mantissa
    code = (y + (bits << (drop - 16)).to(torch.int32)) >> drop
    if least:
        code = torch.maximum(code, (x > 0).to(torch.int32))
    return code, scale


def _adamw_plain(s):
    c, g = s["case"], s["g"].float() * s["clip"]
    eight = c["bits"] == 8
    m = _decode(s["m"], s["ms"]) if eight else s["m"]
    v = _decode(s["v"], s["vs"]) if eight else s["v"]
    p = (s["p"] if s["master"] is None else s["master"]).float()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    root = torch.sqrt(v) * (1 / math.sqrt(1 - BETA2 ** STEP)) + EPS
    p = p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** STEP)) * m / root
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if eight:
        r = _random_bits(g.numel(), s["seed"], g.device)
        code, scale = _encode(m.abs(), r & 0xFFFF, 7, 3, 7, False)
        s["m"].view(torch.uint8).copy_(code | (torch.signbit(m).to(torch.int32) << 7))
        s["ms"].copy_(scale)
        code, scale = _encode(v, r >> 16, 14, 2, 15, True)
        s["v"].view(torch.uint8).copy_(code)
        s["vs"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return {k: s[k] for k in ("p", "master", "m", "v", "ms", "vs") if s[k] is not None}


def run(state):
    op = state["case"]["op"]
    if op == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    if op == "adamw":
        return _adamw_own(state) if own else _adamw_plain(state)
    if own:
        return _framework().grad_norm_clip(state["grads"], 1.0)
    norm = torch.sqrt(state["g"].double().square().sum())
    return torch.stack((norm, torch.clamp(1.0 / (norm + 1e-6), max=1.0))).float()


def work(case):
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "norm":
        rows, cols, e, we = case["rows"], case["cols"], size[case["type"]], size[case["wtype"]]
        stats = rows * 4 * (2 if case["kind"] == "layer" else 1)
        vectors = cols * we * (1 + case["bias"])
        if case["pass"] == "fwd":
            return {"bytes": 2 * rows * cols * e + stats + vectors, "flops": rows * cols * 8}
        return {"bytes": (3 + case["res"]) * rows * cols * e + stats + vectors + cols * we, "flops": rows * cols * 16}
    n = sum(_sizes(case))
    if case["op"] == "clip":
        return {"bytes": n * size[case["gtype"]], "flops": 2 * n}
    p = size[case["ptype"]]
    weights = p + 8 if case["master"] else 2 * p  # a copy in 32 bits is read in the weights' place
    moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * ((n + BLOCK - 1) // BLOCK)
    return {"bytes": n * (weights + size[case["gtype"]]) + moments, "flops": 15 * n}


def _exact_norm(s):
    c = s["case"]
    x, w = s["x"].double(), s["w"].double()
    rows, cols = x.shape
    layer = c["kind"] == "layer"
    if c["pass"] == "fwd":
        mean = x.sum(1) / cols if layer else torch.zeros(rows, dtype=torch.float64, device=x.device)
        centred = x.sub(mean.unsqueeze(1))
        rstd = 1.0 / torch.sqrt((centred ** 2).sum(1) / cols + 1e-5)
        y = torch.einsum("rc,r,c->rc", centred, rstd, w)
        if s["b"] is not None:
            y += s["b"].double()
        return (y, mean, rstd) if layer else (y, rstd)
    dy, rstd = s["dy"].double(), s["rstd"].double()
    # of y = w (x - mean) rstd: the Jacobian is rstd (I - 1 1^T / n - z z^T / n), without the middle term for RMS norm
    z = (x - s["mean"].double().unsqueeze(1)) * rstd.unsqueeze(1)
    up = dy * w
    along = torch.einsum("rc,rc->r", up, z) / cols
    dx = up - along.unsqueeze(1) * z
    if layer:
        dx -= up.sum(1).unsqueeze(1) / cols
    dx *= rstd.unsqueeze(1)
    if s["res"] is not None:
        dx += s["res"].double()
    dw = torch.einsum("rc,rc->c", dy, z)
    if not layer:
        return dx, dw
    return dx, dw, (dy.sum(0) if c["bias"] else None)


def _exact_round(x, u, top, mantissa, smallest):
    """Values of x >= 0 on the 8-bit type's grid, scaled by their blocks, rounded up where the rest plus u reaches one."""
    rows = x.view(-1, BLOCK)
    peak = rows.max(1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(peak > 0, peak, 1.0)))
    e = torch.where(peak < 2.0 ** e, e - 1, e)
    e = torch.clamp(torch.where(peak > 0, e, -1e3), min=top - 126.0)
    t = rows * torch.exp2(top - e)
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(t, min=2.0 ** -300))), min=float(smallest)) - mantissa)
    return (torch.floor(t / unit + u.view(-1, BLOCK)) * unit).view(-1), unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    g = s["g"].double()
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(g)
        return torch.stack((norm, torch.minimum(1.0 / (norm + 1e-6), torch.ones_like(norm))))
    g = g * 0.5
    if case["bits"] == 8:
        m = (s["m"].double().view(-1, BLOCK) * s["ms"].double().unsqueeze(1)).flatten()
        v = (s["v"].double().view(-1, BLOCK) * s["vs"].double().unsqueeze(1)).flatten()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g ** 2 - v)
    old = s["p"].double() if s["master"] is None else s["master"].double()
    step = (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)) ** 0.5 + EPS)
    p = old - LR * DECAY * old - LR * step
    out = {"p": p, "m": m, "v": v}
    if s["master"] is not None:
        out["master"] = p
    if case["bits"] == 8:
        r = _random_bits(g.numel(), s["seed"], g.device)
        q, _ = _exact_round(m.abs(), (r & 0xFFFF).double() / 65536, 7, 3, -6)
        out["m"] = q * torch.where(m < 0, -1.0, 1.0)
        q, _ = _exact_round(v, (r >> 16).double() / 65536, 14, 2, -14)
        out["v"] = torch.where(v > 0, torch.clamp(q, min=2.0 ** -16), q)
        # a block's scale is the power of two below its largest value: next to a border it has no one value
        out["ms"] = out["vs"] = None
    return {k: out[k] for k in ("p", "master", "m", "v", "ms", "vs") if k in out}
