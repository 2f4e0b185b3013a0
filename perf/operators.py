"""Microscaled 4-bit floats: quantising, the linear layer and the expert layer, as timed cases.

Values are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, two codes a byte, the lower nibble first) under a scale per
block of consecutive k:

* ``mx``  blocks of 32, scales are powers of two (e8m0: the byte is the exponent + 127);
* ``nv``  blocks of 16, scales are e4m3, on top of one fp32 scale per tensor.

Three operators:

* ``quant``   rows are quantised and read back (weights when a model is loaded, activations before a product)
* ``linear``  activations are quantised and multiplied with a resident 4-bit weight, with a layer's epilogue
* ``moe``     an expert layer for the few tokens of a decode step: softmax over the router's logits, the top_k
              experts of each token, gate/up with silu(gate) * up, down, weighted sum; 4-bit weights, 16-bit activations

``run`` computes them in elementary torch operations, or with the package's operators where ``own`` is set.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = {"mx": 32, "nv": 16}
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GRID_RMS = 2.93  # of uniformly drawn codes


def listed():
    return [
        # one token's activations on their way into a linear: launches and latency
        dict(name="quant_nv_m1", kind="quant", fmt="nv", dtype="fp16", n=1, k=4096),
        # a prompt of uneven length, bf16 activations
        dict(name="quant_mx_m1733", kind="quant", fmt="mx", dtype="bf16", n=1733, k=11008),
        # a large weight being quantised when the model is loaded
        dict(name="quant_nv_weight", kind="quant", fmt="nv", dtype="fp16", n=28672, k=8192),
        # an attention projection for one sequence
        dict(name="linear_nv_m1", kind="linear", fmt="nv", m=1, k=4096, n=4096, epilogue="none"),
        # an output projection whose width is no multiple of a tile, for a few sequences
        dict(name="linear_mx_m7_ragged", kind="linear", fmt="mx", m=7, k=4096, n=32016, epilogue="bias"),
        # a down projection with the residual added, at a serving batch
        dict(name="linear_nv_m48", kind="linear", fmt="nv", m=48, k=28672, n=8192, epilogue="residual"),
        # a prompt of uneven length through an MLP's first linear
        dict(name="linear_mx_m333", kind="linear", fmt="mx", m=333, k=4096, n=11008, epilogue="bias_silu"),
        # a 2048-token prompt through a fused gate/up projection
        dict(name="linear_nv_m2048", kind="linear", fmt="nv", m=2048, k=4096, n=22016, epilogue="none"),
        # the longest prompt and the largest linear
        dict(name="linear_mx_m4096", kind="linear", fmt="mx", m=4096, k=8192, n=28672, epilogue="none"),
        # a decode step of one sequence and of eight through eight large experts
        dict(name="moe_mx_t1", kind="moe", fmt="mx", tokens=1, hidden=4096, ffn=14336, experts=8, top_k=2),
        dict(name="moe_nv_t8", kind="moe", fmt="nv", tokens=8, hidden=4096, ffn=14336, experts=8, top_k=2),
        # many small experts, most of them with a token or two
        dict(name="moe_mx_t29_small", kind="moe", fmt="mx", tokens=29, hidden=2048, ffn=1408, experts=64, top_k=6),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, round(v / step) * step))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "moe", "moe"])
    fmt = rng.choice(["mx", "nv"])
    if kind == "quant":
        k = _log_int(rng, 256, 28672, 32)
        return dict(kind=kind, fmt=fmt, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    n=_log_int(rng, 1, min(32768, 28672 * 4096 // k)), k=k)
    if kind == "linear":
        k = _log_int(rng, 512, 28672, rng.choice([32, 128]))
        n = _log_int(rng, 256, min(32768, 28672 * 8192 // k), rng.choice([1, 16, 128]))
        return dict(kind=kind, fmt=fmt, m=_log_int(rng, 1, 4096), k=k, n=n,
                    epilogue=rng.choice(["none", "bias", "bias_silu", "residual"]))
    while True:
        c = dict(kind=kind, fmt=fmt, tokens=_log_int(rng, 1, 32), hidden=_log_int(rng, 512, 7168, 64),
                 ffn=_log_int(rng, 256, 14336, 64), experts=rng.choice([4, 8, 16, 32, 64, 128]), top_k=rng.choice([1, 2, 4, 6, 8]))
        if c["top_k"] <= c["experts"] and c["experts"] * c["hidden"] * c["ffn"] <= 8 * 4096 * 14336:
            return c


# ------------------------------------------------------------------ inputs

def _activations(g, m, k, dtype=torch.float16):
    # a few channels are much larger than the rest, as in the residual stream of a trained model
    gain = torch.exp(0.7 * torch.randn(k, device=DEV, generator=g))
    return (torch.randn(m, k, device=DEV, generator=g) * gain).to(dtype)


def _weight(g, fmt, n, k, experts=None):
    """Codes uint8 [(experts,) n, k / 2], scales uint8 [(experts,) n, k / block], tensor scales fp32 or None; sums over
    k are of order one."""
    lead = () if experts is None else (experts,)
    codes = torch.randint(0, 256, lead + (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    size = 1.0 / (GRID_RMS * math.sqrt(k))
    shape = lead + (n, k // BLOCK[fmt])
    if fmt == "mx":
        mid = 127 + round(math.log2(size))
        return codes, torch.randint(mid - 1, mid + 2, shape, dtype=torch.uint8, device=DEV, generator=g), None
    # e4m3 from 64 to 448 (0x68 to 0x7e), under a tensor scale
    scales = torch.randint(0x68, 0x7f, shape, dtype=torch.uint8, device=DEV, generator=g)
    ts = (0.5 + torch.rand(lead or (1,), device=DEV, generator=g)) * (size / 200.0)
    return codes, scales, ts


def _own_scales(scales):
    if not own:
        return None
    from relax_b200 import ops
    return ops.preprocess_fp4_scales(scales)


def _tensor_scale(x):
    return (x.abs().amax().float() / (448.0 * 6.0)).reshape(1)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "quant":
        s["x"] = _activations(g, c["n"], c["k"], DTYPES[c["dtype"]])
        s["ts"] = _tensor_scale(s["x"]) if c["fmt"] == "nv" else None
    elif c["kind"] == "linear":
        s["x"] = _activations(g, c["m"], c["k"])
        s["ts"] = _tensor_scale(s["x"]) if c["fmt"] == "nv" else None
        s["w"], s["ws"], s["wts"] = _weight(g, c["fmt"], c["n"], c["k"])
        s["ws_own"] = _own_scales(s["ws"])
        s["bias"] = torch.randn(c["n"], device=DEV, generator=g).half() if c["epilogue"] in ("bias", "bias_silu") else None
        s["residual"] = torch.randn(c["m"], c["n"], device=DEV, generator=g).half() if c["epilogue"] == "residual" else None
    else:
        h, f, e = c["hidden"], c["ffn"], c["experts"]
        s["x"] = torch.randn(c["tokens"], h, device=DEV, generator=g).half()
        s["logits"] = 2.0 * torch.randn(c["tokens"], e, device=DEV, generator=g)
        s["w1"], s["s1"], s["ts1"] = _weight(g, c["fmt"], 2 * f, h, e)  # gate rows, then up rows
        s["w2"], s["s2"], s["ts2"] = _weight(g, c["fmt"], h, f, e)
        s["s1_own"], s["s2_own"] = _own_scales(s["s1"]), _own_scales(s["s2"])
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"quant": _own_quant, "linear": _own_linear, "moe": _own_moe}[kind](state)
    return {"quant": _plain_quant, "linear": _plain_linear, "moe": _plain_moe}[kind](state)


def _own_quant(s):
    from relax_b200 import ops
    fmt = s["case"]["fmt"]
    codes, scales = ops.encode_fp4(s["x"], fmt, tensor_scale=s["ts"])
    return ops.decode_fp4(codes, scales, fmt, tensor_scale=s["ts"], dtype=s["x"].dtype)


def _own_linear(s):
    from relax_b200 import ops
    c = s["case"]
    return ops.linear_fp4(s["x"], s["w"], s["ws_own"], c["fmt"], x_tensor_scale=s["ts"], w_tensor_scale=s["wts"],
                          bias=s["bias"], residual=s["residual"],
                          activation="silu" if c["epilogue"] == "bias_silu" else "identity",
                          binary_op="plus" if c["epilogue"] == "residual" else "")


def _own_moe(s):
    from relax_b200 import ops
    c = s["case"]
    return ops.moe_layer_fp4(s["x"], s["logits"], s["w1"], s["s1_own"], s["w2"], s["s2_own"], c["top_k"], c["fmt"],
                             gate_up_tensor_scale=s["ts1"], down_tensor_scale=s["ts2"], renormalize=True)


def _values(codes):
    """e2m1 codes, two a byte -> fp32 values."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    return grid[nibbles.int()]


def _scale_values(scales, fmt):
    if fmt == "mx":
        return torch.exp2(scales.float() - 127.0)
    exponent, mantissa = (scales >> 3).float(), (scales & 7).float()
    return torch.where(exponent > 0, torch.exp2(exponent - 7.0) * (1.0 + mantissa / 8.0), mantissa * 2.0 ** -9)


def _dequantised(codes, scales, fmt, ts):
    """fp32 values of a quantised matrix [n, k]."""
    v = _values(codes).unflatten(-1, (-1, BLOCK[fmt])) * _scale_values(scales, fmt).unsqueeze(-1)
    return v.flatten(-2) if ts is None else v.flatten(-2) * ts


def _quantised(x, fmt, ts):
    """(fp32 values on the e2m1 grid [n, blocks, block], fp32 block scales [n, blocks]).  Quotients by a tensor scale are
    taken in 64 bits: what lies next to the border between two codes would fall on either side in 32."""
    blocks = x.float().unflatten(-1, (-1, BLOCK[fmt]))
    amax = blocks.abs().amax(-1)
    if fmt == "mx":
        exponent = torch.frexp(amax).exponent.float() - 3.0  # floor(log2(amax)) - 2
        scale = torch.exp2(torch.where(amax > 0, exponent, -127.0).clamp_min(-127.0))
        mag = blocks.abs() / scale.unsqueeze(-1)
    else:
        r = amax.double() / (6.0 * ts.double())
        quantum = torch.exp2((torch.frexp(r).exponent - 1).clamp_min(-6).double() - 3.0)
        scale = (torch.round(r / quantum) * quantum).clamp_max(448.0)  # torch.round: ties to even
        mag = torch.where(scale.unsqueeze(-1) > 0, blocks.abs().double() / (scale * ts.double()).unsqueeze(-1), 0.0)
    # ties go to the even code
    steps = ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False), (1.75, 0.5, True),
             (2.5, 1.0, False), (3.5, 1.0, True), (5.0, 2.0, False))
    q = torch.zeros_like(blocks)
    for border, step, up in steps:
        q += ((mag >= border) if up else (mag > border)).float() * step
    return torch.copysign(q, blocks), scale.float()


def _plain_quant(s):
    q, scale = _quantised(s["x"], s["case"]["fmt"], s["ts"])
    v = (q * scale.unsqueeze(-1)).flatten(-2)
    return (v if s["ts"] is None else v * s["ts"]).to(s["x"].dtype)


def _plain_linear(s):
    c = s["case"]
    q, scale = _quantised(s["x"], c["fmt"], s["ts"])
    a = (q * scale.unsqueeze(-1)).flatten(-2)
    y = a @ _dequantised(s["w"], s["ws"], c["fmt"], None).T
    if s["ts"] is not None:
        y = y * (s["ts"] * s["wts"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["epilogue"] == "bias_silu":
        y = y / (1.0 + torch.exp(-y))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.half()


def _plain_moe(s):
    c = s["case"]
    f, fmt = c["ffn"], c["fmt"]
    x = s["x"].float()
    weight = torch.exp(s["logits"] - s["logits"].amax(-1, keepdim=True))
    order = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]
    gates = torch.zeros_like(weight).scatter_(1, order, weight.gather(1, order))
    gates = gates / gates.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(c["experts"]):
        ts1, ts2 = (None, None) if fmt == "mx" else (s["ts1"][e], s["ts2"][e])
        gu = x @ _dequantised(s["w1"][e], s["s1"][e], fmt, ts1).T
        h = gu[:, :f] / (1.0 + torch.exp(-gu[:, :f])) * gu[:, f:]
        out += gates[:, e:e + 1] * (h @ _dequantised(s["w2"][e], s["s2"][e], fmt, ts2).T)
    return out.half()


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_decoded(codes, scales, fmt, ts):
    low, high = (codes % 16).long(), torch.div(codes, 16, rounding_mode="floor").long()
    nib = torch.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), dtype=torch.long, device=codes.device)
    nib[..., 0::2], nib[..., 1::2] = low, high
    m = (nib % 8).double()
    v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8)) * (1.0 - 2.0 * (nib >= 8).double())
    b = scales.double()
    if fmt == "mx":
        sc = torch.pow(2.0, b - 127.0)
    else:
        e = torch.floor(b / 8)
        sc = torch.where(e == 0, (b - 8 * e) / 512.0, (8 + b - 8 * e) * torch.pow(2.0, e - 10.0))
    out = v * sc.repeat_interleave(BLOCK[fmt], dim=-1)
    return out if ts is None else out * ts.double()


def _exact_quantised(x, fmt, ts):
    n, k = x.shape
    y = x.double().view(n, k // BLOCK[fmt], BLOCK[fmt])
    top = y.abs().max(dim=-1, keepdim=True).values
    if fmt == "mx":
        # the largest power of two that is not above the maximum, over four
        p = torch.pow(2.0, torch.floor(torch.log2(top.clamp_min(2.0 ** -200))))
        p = torch.where(p > top, p / 2, torch.where(2 * p <= top, 2 * p, p))
        unit = (p / 4).clamp_min(2.0 ** -127)
    else:
        want = top / 6.0 / ts.double()
        lo = torch.pow(2.0, torch.floor(torch.log2(want.clamp_min(2.0 ** -6))).clamp(-6, 8)) / 8.0
        unit = torch.minimum(torch.round(want / lo) * lo, torch.full_like(want, 448.0)) * ts.double()
    z = torch.where(unit > 0, y / torch.where(unit > 0, unit, 1.0), 0.0)
    a = z.abs()
    # spacing 1/2 below 2, 1 below 4, 2 above; torch.round settles ties to even, which is the even code
    r = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2))).clamp_max(6.0)
    return (torch.sign(z) * r * unit).view(n, k)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    fmt = c["fmt"]
    if c["kind"] == "quant":
        return _exact_quantised(s["x"], fmt, s["ts"])
    if c["kind"] == "linear":
        y = _exact_quantised(s["x"], fmt, s["ts"]) @ _exact_decoded(s["w"], s["ws"], fmt, s["wts"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if c["epilogue"] == "bias_silu":
            y = y * torch.sigmoid(y)
        return y if s["residual"] is None else y + s["residual"].double()
    f = c["ffn"]
    x, logits = s["x"].double(), s["logits"].double()
    out = torch.zeros_like(x)
    # rank of an expert for a token: those with larger logits, and equal ones before it
    before = torch.arange(c["experts"], device=DEV)
    ahead = (logits.unsqueeze(1) > logits.unsqueeze(2)) | ((logits.unsqueeze(1) == logits.unsqueeze(2))
                                                          & (before.view(1, 1, -1) < before.view(1, -1, 1)))
    chosen = (ahead.sum(-1) < c["top_k"]).double()
    p = torch.softmax(logits, dim=-1) * chosen
    p = p / p.sum(-1, keepdim=True)
    for e in range(c["experts"]):
        ts1, ts2 = (None, None) if fmt == "mx" else (s["ts1"][e], s["ts2"][e])
        gu = x @ _exact_decoded(s["w1"][e], s["s1"][e], fmt, ts1).t()
        h = gu[:, :f] * torch.sigmoid(gu[:, :f]) * gu[:, f:]
        out += p[:, e:e + 1] * (h @ _exact_decoded(s["w2"][e], s["s2"][e], fmt, ts2).t())
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def _bytes_of(n, k, fmt):
    return n * k / 2 + n * k / BLOCK[fmt]


def work(case):
    c = case
    fmt = c["fmt"]
    if c["kind"] == "quant":
        width = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": 2.0 * width * c["n"] * c["k"], "flops": 0}
    if c["kind"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        b = 2.0 * m * k + _bytes_of(n, k, fmt) + 2.0 * m * n
        b += 2.0 * n * (c["epilogue"] in ("bias", "bias_silu")) + 2.0 * m * n * (c["epilogue"] == "residual")
        return {"bytes": b, "flops": 2.0 * m * n * k}
    h, f, t, e = c["hidden"], c["ffn"], c["tokens"], c["experts"]
    # experts that some token chooses, under an even spread: only their weights are needed
    used = e * (1.0 - (1.0 - c["top_k"] / e) ** t)
    return {"bytes": used * (_bytes_of(2 * f, h, fmt) + _bytes_of(h, f, fmt)) + t * (4.0 * h + 4.0 * e),
            "flops": 6.0 * t * c["top_k"] * h * f}
