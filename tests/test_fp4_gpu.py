"""Microscaled 4-bit floats on the GPU against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import relax_b200
from relax_b200 import ops
from tests import fp4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _np(t):
    return t.detach().double().cpu().numpy()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _check_encode(x, fmt, ts=None):
    t = None if ts is None else torch.tensor([ts], device="cuda", dtype=torch.float32)
    codes, scales = ops.encode_fp4(x, fmt, tensor_scale=t)
    want_c, want_s = ref.encode(_np(x), fmt, 1.0 if ts is None else float(np.float32(ts)))
    got_s = scales.cpu().numpy()
    assert np.array_equal(got_s, ref.tile(want_s)), "scales (zero past the matrix)"
    assert np.array_equal(codes.cpu().numpy(), want_c), "codes"
    return codes, scales, want_c, want_s


# ------------------------------------------------------------------ quantising

@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n, k", [(1, 32), (1, 4096), (3, 64), (127, 96), (128, 512), (129, 544), (200, 1056)])
def test_encode(fmt, dtype, n, k):
    g = _gen(n * k)
    x = (torch.randn(n, k, device="cuda", generator=g) * torch.exp(3 * torch.randn(n, k, device="cuda", generator=g))).to(TYPES[dtype])
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    x[0, :32] = 0
    _check_encode(x, fmt)
    if fmt == "nv":
        for ts in (0.25, 0.0123456, 3.7e-5, 1.0 / 3.0):
            _check_encode(x, fmt, ts)


@pytest.mark.parametrize("ts", [None, 0.5, 0.1, 1.7e-3])
def test_encode_borders(ts):
    """Elements on the borders between codes, one unit of fp32 beside them, and block maxima on the borders between scales."""
    unit = np.float32(1.0 if ts is None else ts)
    v = ref.e4m3_bytes()
    rows = []
    for b in list(range(1, 0x7f, 3)) + [0x7e]:
        amax = np.float32(6 * v[b] * unit)
        border = ((ref.GRID[:-1] + ref.GRID[1:]) / 2 * v[b] * unit).astype(np.float32)
        rows.append(np.concatenate([[amax, -amax], border, -border]).astype(np.float32))
        rows.append(np.concatenate([[amax, 0], np.nextafter(border, np.float32(1e9)), np.nextafter(border, np.float32(-1e9))]).astype(np.float32))
    for i in range(0x7e):
        mid = np.float32((v[i] + v[i + 1]) / 2 * 6 * unit)
        for m in (mid, np.nextafter(mid, np.float32(1e9)), np.nextafter(mid, np.float32(0))):
            rows.append(np.concatenate([[m], np.zeros(15)]).astype(np.float32))
    x = np.stack(rows)
    x = np.concatenate([x, x[::-1]], axis=1)
    _check_encode(torch.from_numpy(x).cuda(), "nv", ts)
    y = x.astype(np.float16).astype(np.float32)
    _check_encode(torch.from_numpy(y).cuda().half(), "nv", ts)


def test_encode_mx_borders():
    rows = []
    for e in (-149, -130, -127, -126, -125, -124, -20, 0, 3, 100, 127):
        one = np.float64(2.0) ** e
        rows.append(np.concatenate([[one * 1.9999999], np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]) * one / 4, np.zeros(23)]))
    x = np.stack(rows).astype(np.float32)
    x[~np.isfinite(x)] = np.float32(3.4e38)
    _check_encode(torch.from_numpy(x).cuda(), "mx")


@pytest.mark.parametrize("ts", [0.0, -1.0, float("nan"), float("inf"), 1e-38, 3e38, 1e-44])
def test_encode_odd_tensor_scales(ts):
    x = torch.randn(5, 64, device="cuda", generator=_gen(1))
    x[1] *= 1e-37
    x[2] *= 1e30
    _check_encode(x, "nv", ts)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_encode_not_finite(fmt):
    x = torch.randn(4, 128, device="cuda", generator=_gen(2))
    x[0, 3], x[1, 40], x[2, 127] = float("inf"), float("nan"), float("-inf")
    codes, scales, _, _ = _check_encode(x.half(), fmt)
    y = ops.decode_fp4(codes, scales, fmt, dtype=torch.float32)
    block = ref.BLOCK[fmt]
    for r, c in ((0, 3), (1, 40), (2, 127)):
        b = c // block * block
        assert torch.isnan(y[r, b:b + block]).all()
        y[r, b:b + block] = 0
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_encode_strides_and_batches(fmt):
    g = _gen(5)
    wide = torch.randn(70, 256, device="cuda", generator=g).half()
    a = ops.encode_fp4(wide[:, 64:192], fmt)         # rows of a wider matrix
    b = ops.encode_fp4(wide[:, 64:192].contiguous(), fmt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = wide.t()[:, :64]                             # the other order
    a, b = ops.encode_fp4(t, fmt), ops.encode_fp4(t.contiguous(), fmt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    flat = torch.randn(70 * 64 + 1, device="cuda", generator=g).half()[1:]
    a, b = ops.encode_fp4(flat.view(70, 64), fmt), ops.encode_fp4(flat.clone().view(70, 64), fmt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = torch.randn(3, 130, 96, device="cuda", generator=g).half()
    ts = torch.tensor([0.5, 0.01, 7.0], device="cuda") if fmt == "nv" else None
    codes, scales = ops.encode_fp4(x, fmt, tensor_scale=ts)
    y = ops.decode_fp4(codes, scales, fmt, tensor_scale=ts, dtype=torch.float32)
    for e in range(3):
        te = ts[e:e + 1] if ts is not None else None
        c, s = ops.encode_fp4(x[e], fmt, tensor_scale=te)
        assert torch.equal(c, codes[e]) and torch.equal(s, scales[e])
        assert torch.equal(ops.decode_fp4(c, s, fmt, tensor_scale=te, dtype=torch.float32), y[e])
    c, s = ops.encode_fp4(x[:, :0], fmt, tensor_scale=ts)
    assert c.shape == (3, 0, 48) and s.numel() == 0


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_decode(fmt, dtype):
    """Every code under every scale byte; one rounding (two in nv: the tensor scale's in fp32, then the type's)."""
    g = _gen(7)
    codes = torch.arange(256, device="cuda").repeat(256, 1).to(torch.uint8)
    scales = torch.arange(256, device="cuda").view(256, 1).expand(256, 512 // ref.BLOCK[fmt]).to(torch.uint8)
    if fmt == "nv":
        scales = scales & 0x7f
    ts = torch.rand(1, device="cuda", generator=g) if fmt == "nv" else None
    y = _np(ops.decode_fp4(codes, ops.preprocess_fp4_scales(scales), fmt, tensor_scale=ts, dtype=TYPES[dtype]))
    want = ref.decode(codes.cpu().numpy(), scales.cpu().numpy(), fmt, 1.0 if ts is None else float(ts))
    info = torch.finfo(TYPES[dtype])
    step = np.maximum(np.abs(want), info.tiny) * (info.eps / 2 + (2.0 ** -24 if fmt == "nv" else 0.0))
    big = np.abs(want) > info.max * (1 - info.eps / 4)
    assert np.array_equal(np.isnan(y), np.isnan(want))
    assert (np.isinf(y) | (np.abs(y) == info.max) | ~big)[~np.isnan(want)].all()
    fine = ~np.isnan(want) & ~big
    assert (np.abs(y - want)[fine] <= step[fine] + info.tiny * info.eps).all()


@pytest.mark.parametrize("rows, blocks", [(1, 1), (31, 3), (128, 4), (129, 9), (300, 16)])
def test_scale_tiles(rows, blocks):
    s = torch.randint(0, 256, (2, rows, blocks), dtype=torch.uint8, device="cuda", generator=_gen(rows))
    got = ops.preprocess_fp4_scales(s).cpu().numpy()
    for e in range(2):
        assert np.array_equal(got[e], ref.tile(s[e].cpu().numpy()))
    as_float = s.view(torch.float8_e4m3fn)
    assert torch.equal(ops.preprocess_fp4_scales(as_float).cpu(), torch.from_numpy(got))


# ------------------------------------------------------------------ products

def _operand(g, fmt, rows, k):
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    lo, hi = (120, 132) if fmt == "mx" else (0x20, 0x50)
    scales = torch.randint(lo, hi, (rows, k // ref.BLOCK[fmt]), dtype=torch.uint8, device="cuda", generator=g)
    return codes, ops.preprocess_fp4_scales(scales), ref.decode(codes.cpu().numpy(), scales.cpu().numpy(), fmt)


def _check_product(got, a, w, alpha=1.0, tail=None):
    info = torch.finfo(got.dtype)
    err, half = ref.gemm_bound(a, w, info.eps)
    exact = (a @ w.T) * alpha
    err = err * abs(alpha) + 2.0 ** -23 * np.abs(exact)  # the tensor scales' product, and its product with the sum
    if tail is not None:
        exact, err = tail(exact, err)
    got = _np(got)
    # a value at least half a step above the largest number rounds to infinity, and either is right within err of that border
    top = info.max * (1 + info.eps / 4)
    over = np.abs(exact) >= top - err
    fine = np.isinf(got) & (np.sign(got) == np.sign(exact)) | (np.abs(got) == info.max) & (np.abs(exact) < top + err)
    got = np.where(over & fine, exact, got)
    off = np.abs(got - exact) - err - half * (np.abs(exact) + err) - info.tiny * info.eps
    bad = np.argwhere(~(off <= 0))
    assert bad.size == 0, (len(bad), bad[:5], got[tuple(bad[0])], exact[tuple(bad[0])])


SHAPES = [(1, 1, 32), (1, 128, 64), (3, 130, 96), (8, 256, 256), (16, 64, 288), (17, 200, 320), (33, 127, 512), (64, 384, 1056),
          (100, 129, 2080), (129, 256, 800), (200, 100, 256), (257, 300, 544), (520, 257, 1024), (1, 4096, 4096), (40, 96, 8192),
          (1000, 513, 96), (300, 9600, 64), (1300, 4100, 288), (385, 1024, 1536), (256, 128, 32),
          (70, 300, 4096), (128, 257, 8224), (333, 2600, 3104), (600, 9500, 2592)]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m, n, k", SHAPES)
def test_gemm(fmt, m, n, k):
    g = _gen(m * 7 + n * 3 + k)
    (ac, asc, a), (wc, wsc, w) = _operand(g, fmt, m, k), _operand(g, fmt, n, k)
    _check_product(ops.gemm_fp4(ac, asc, wc, wsc, fmt, dtype=torch.float32), a, w)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_gemm_every_code_and_scale(fmt):
    """One product per output: row i of w holds one code under one scale, a one-hot row of a picks it."""
    k = 512
    block = ref.BLOCK[fmt]
    a = np.zeros((k, k), dtype=np.uint8)
    np.fill_diagonal(a, 2)  # the code of 1
    ac = torch.from_numpy(a[:, 0::2] | (a[:, 1::2] << 4)).cuda()
    asc = ops.preprocess_fp4_scales(torch.full((k, k // block), 127 if fmt == "mx" else 0x38, dtype=torch.uint8, device="cuda"))
    g = _gen(11)
    wc, wsc, w = _operand(g, fmt, 256, k)
    out = ops.gemm_fp4(ac, asc, wc, wsc, fmt, dtype=torch.float32)
    assert np.array_equal(_np(out).T, w), "products of one by every element, exactly"


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m, n", [(5, 136), (70, 131), (300, 264), (150, 131)])
def test_gemm_epilogue(fmt, dtype, m, n):
    k, t = 256, TYPES[dtype]
    g = _gen(m + n if m < 100 else 5)
    (ac, asc, a), (wc, wsc, w) = _operand(g, fmt, m, k), _operand(g, fmt, n, k)
    scale = 1.0 / 64
    ta = torch.tensor([scale], device="cuda") if fmt == "nv" else None
    tw = torch.tensor([0.3], device="cuda") if fmt == "nv" else None
    alpha = scale * float(np.float32(0.3)) if fmt == "nv" else 1.0
    bias = torch.randn(n, device="cuda", generator=g).to(t)
    res = torch.randn(m, n, device="cuda", generator=g).to(t)
    b, r = _np(bias), _np(res)

    def relu(y):
        return np.maximum(y, 0)

    def silu(y):
        return y / (1 + np.exp(-np.clip(y, -700, 700)))

    def gelu(y):
        from scipy.special import erf
        return 0.5 * y * (1 + erf(y / np.sqrt(2)))

    acts = {"identity": lambda y: y, "relu": relu, "silu": silu, "gelu": gelu}
    for act, bin_, un in (("identity", "", "identity"), ("relu", "", "identity"), ("silu", "plus", "identity"),
                          ("gelu", "multiply", "relu"), ("identity", "multiply", "identity"), ("silu", "", "relu")):
        got = ops.gemm_fp4(ac, asc, wc, wsc, fmt, ta, tw, bias=bias, residual=res if bin_ else None, activation=act,
                           binary_op=bin_, unary_op=un, dtype=t)

        def tail(y, err):
            # the bias is one more fp32 addition; |activation'| <= 1.13; its own evaluation in fp32 (exp, erf, a division)
            # is good to 2^-20 of its input, the residual one more operation
            y = y + b
            err = err + 2.0 ** -24 * np.abs(y)
            z = acts[act](y)
            err = 1.13 * err + 2.0 ** -20 * np.abs(y)
            if bin_ == "plus":
                z, err = z + r, err + 2.0 ** -24 * np.abs(z + r)
            if bin_ == "multiply":
                z, err = z * r, err * np.abs(r) + 2.0 ** -24 * np.abs(z * r)
            return (np.maximum(z, 0) if un == "relu" else z), err

        _check_product(got, a, w, alpha, tail)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_gemm_keeps_a_bad_row_to_itself(fmt):
    g = _gen(3)
    x = torch.randn(40, 512, device="cuda", generator=g).half()
    w = torch.randn(200, 512, device="cuda", generator=g).half()
    ac, asc = ops.encode_fp4(x, fmt)
    wc, wsc = ops.encode_fp4(w, fmt)
    base = ops.gemm_fp4(ac, asc, wc, wsc, fmt)
    x[7, 100] = float("inf")
    w[150, 5] = float("nan")
    ac, asc = ops.encode_fp4(x, fmt)
    wc, wsc = ops.encode_fp4(w, fmt)
    out = ops.gemm_fp4(ac, asc, wc, wsc, fmt)
    assert torch.isnan(out[7]).all() and torch.isnan(out[:, 150]).all()
    out[7], out[:, 150] = base[7], base[:, 150]
    assert torch.equal(out, base)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m, n, k, dtype", [(1, 512, 1024, "fp16"), (2, 4096, 4096, "bf16"), (9, 300, 544, "bf16"), (16, 130, 2080, "fp32"), (13, 257, 32, "fp16"), (17, 300, 544, "fp16"), (65, 129, 96, "fp16"), (300, 256, 2048, "fp32")])
def test_linear(fmt, m, n, k, dtype):
    g = _gen(m + n + k)
    x = (torch.randn(m, k, device="cuda", generator=g) * torch.exp(torch.randn(k, device="cuda", generator=g))).to(TYPES[dtype])
    wc, wsc, w = _operand(g, fmt, n, k)
    ts = (x.abs().amax().float() / 2688).reshape(1) if fmt == "nv" else None
    tsv = 1.0 if ts is None else float(ts)
    out = ops.linear_fp4(x, wc, wsc, fmt, x_tensor_scale=ts)
    assert out.dtype == x.dtype
    c, s = ref.encode(_np(x), fmt, tsv)
    a = ref.decode(c, s, fmt)
    _check_product(out, a, w, tsv)
    # the same in two steps, a batch of the same rows, and rows in place
    ac, asc = ops.encode_fp4(x, fmt, tensor_scale=ts)
    assert torch.equal(ops.gemm_fp4(ac, asc, wc, wsc, fmt, a_tensor_scale=ts, dtype=x.dtype), out)
    assert torch.equal(ops.linear_fp4(x.view(1, m, k), wc, wsc, fmt, x_tensor_scale=ts), out.view(1, m, n))
    ws = torch.empty(ops.linear_fp4_workspace_bytes(m, k, fmt), dtype=torch.uint8, device="cuda")
    given = torch.empty_like(out)
    assert ops.linear_fp4(x, wc, wsc, fmt, x_tensor_scale=ts, workspace=ws, out=given) is given
    assert torch.equal(given, out)


def test_empty_batch():
    wc, wsc, _ = _operand(_gen(0), "mx", 64, 64)
    assert ops.linear_fp4(torch.empty(0, 64, device="cuda").half(), wc, wsc, "mx").shape == (0, 64)


def test_linear_in_a_graph_and_on_streams():
    g = _gen(21)
    layers = [_operand(g, "nv", 512, 512)[:2] for _ in range(3)]
    x = torch.randn(6, 512, device="cuda", generator=g).half()
    ts = torch.tensor([0.01], device="cuda")

    def chain(x):
        for c, s in layers:
            x = ops.linear_fp4(x, c, s, "nv", x_tensor_scale=ts, w_tensor_scale=ts)
        return x

    want = chain(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [chain(x) for _ in range(20)]
    here = [chain(x) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got + here)
    before = relax_b200.get_launch_overlap()
    for overlap in (False, True):
        relax_b200.set_launch_overlap(overlap)
        try:
            graph = torch.cuda.CUDAGraph()
            buf = x.clone()
            with torch.cuda.graph(graph):
                out = chain(buf)
        finally:
            relax_b200.set_launch_overlap(before)
        for i in range(20):
            buf.copy_(x if i % 2 else -x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, chain(x if i % 2 else -x))
