"""Linears in 4-bit floats of more than 64 rows where tiles are few (two pairs of CTAs share k) and where a pair has several, with
every epilogue; the quantiser at the sizes where a warp's rows change."""
import numpy as np
import pytest
import torch

from relax_b200 import ops
from tests import fp4_ref as ref
from tests.test_fp4_gpu import TYPES, _check_encode, _check_product, _gen, _np, _operand

pytestmark = pytest.mark.gpu


def _epilogue(act, bin_, b, r):
    """What the sums go through, and its error: the bias is one fp32 addition, |activation'| <= 1.13, the activation itself is good
    to 2^-20 of its input, the residual one more operation."""
    def tail(y, err):
        if b is not None:
            y = y + b
            err = err + 2.0 ** -24 * np.abs(y)
        if act == "silu":
            z = y / (1 + np.exp(-np.clip(y, -700, 700)))
            err = 1.13 * err + 2.0 ** -20 * np.abs(y)
        else:
            z = np.maximum(y, 0) if act == "relu" else y
        if bin_ == "plus":
            z, err = z + r, err + 2.0 ** -24 * np.abs(z + r)
        if bin_ == "multiply":
            z, err = z * r, err * np.abs(r) + 2.0 ** -24 * np.abs(z * r)
        return z, err
    return tail


# (k 4096 and above with at most 33 tiles of 256 x 256 is shared by two pairs; 9504 and 4104 columns leave a pair several tiles)
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m, n, k", [(65, 264, 4096), (97, 131, 4128), (130, 520, 4160), (257, 136, 4096), (300, 1000, 6176),
                                     (270, 9504, 96), (1290, 4104, 64), (900, 6001, 32)])
@pytest.mark.parametrize("act, bin_", [("silu", "plus"), ("identity", "multiply"), ("relu", ""), ("identity", "plus")])
def test_epilogues_of_large_batches(fmt, dtype, m, n, k, act, bin_):
    t, g = TYPES[dtype], _gen(m + n + k)
    (ac, asc, a), (wc, wsc, w) = _operand(g, fmt, m, k), _operand(g, fmt, n, k)
    scale = 2.0 ** -10  # keeps the sums of 6176 products inside fp16
    ta = torch.tensor([scale], device="cuda") if fmt == "nv" else None
    if fmt == "mx":
        wsc = ops.preprocess_fp4_scales(torch.full((n, k // 32), 118, dtype=torch.uint8, device="cuda"))
        w = ref.decode(wc.cpu().numpy(), np.full((n, k // 32), 118, dtype=np.uint8), fmt)
    bias = torch.randn(n, device="cuda", generator=g).to(t) if act != "identity" else None
    res = torch.randn(m, n, device="cuda", generator=g).to(t) if bin_ else None
    got = ops.gemm_fp4(ac, asc, wc, wsc, fmt, ta, None, bias=bias, residual=res, activation=act, binary_op=bin_, dtype=t)
    _check_product(got, a, w, scale if fmt == "nv" else 1.0,
                   _epilogue(act, bin_, None if bias is None else _np(bias), None if res is None else _np(res)))


@pytest.mark.parametrize("m, k", [(80, 4096), (600, 64)])
def test_residual_with_and_without_alignment(m, k):
    """The same numbers whether the residual comes in 16-byte pieces or element by element, and in place."""
    g, n = _gen(m), 9504 if k == 64 else 264
    (ac, asc, _), (wc, wsc, _) = _operand(g, "mx", m, k), _operand(g, "mx", n, k)
    base = torch.randn(m * n + 8, device="cuda", generator=g, dtype=torch.float32).half()
    aligned = base[:m * n].view(m, n)
    odd = base[1:m * n + 1].view(m, n)
    odd.copy_(aligned.clone())
    want = ops.gemm_fp4(ac, asc, wc, wsc, "mx", residual=odd, binary_op="plus")
    plain = odd.clone()
    assert torch.equal(ops.gemm_fp4(ac, asc, wc, wsc, "mx", residual=plain, binary_op="plus"), want)
    assert torch.equal(ops.gemm_fp4(ac, asc, wc, wsc, "mx", residual=plain, binary_op="plus", out=plain), want)
    assert torch.equal(plain, want)


@pytest.mark.parametrize("m, k", [(3, 256), (80, 4096), (300, 96)])
def test_silu_over_its_range(m, k):
    """Products of nothing: the result is silu of the bias, from one end of fp32 to the other."""
    v = [0.0, 1e-30, 1e-5, 0.3, 1.0, 5.0, 20.0, 87.0, 88.5, 90.0, 104.0, 1e3, 1e10, 3e38]
    bias = torch.tensor(v + [-x for x in v], device="cuda")
    n = bias.numel()
    zero = lambda rows: (torch.zeros(rows, k // 2, dtype=torch.uint8, device="cuda"),
                         ops.preprocess_fp4_scales(torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda")))
    got = _np(ops.gemm_fp4(*zero(m), *zero(n), "mx", bias=bias, activation="silu", dtype=torch.float32))
    b = _np(bias)
    want = np.where(b > -700, b / (1 + np.exp(-np.maximum(b, -700))), 0.0)
    # 2^-20 of the input, and of the result |b| 2^-22 (the exponent's rounding).  1 / (1 + exp(-b)) below 2^-126, the smallest
    # normal number, is 0, which takes up to |b| 2^-126 away: -88.5 / (1 + exp(88.5)) = -3.3e-37 becomes 0, 88.5 * 2^-126 = 1.04e-36.
    tol = 2.0 ** -20 * np.minimum(np.abs(b), np.maximum(np.abs(want) * (1 + np.abs(b)), 1e-37))
    assert (np.abs(got - want) <= np.maximum(tol, np.minimum(np.abs(b), 104.0) * 2.0 ** -126)).all()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("n, k", [(47, 12000), (250, 14368), (520, 8224), (1100, 4096), (2000, 4128)])
def test_encode_at_rows_of_a_warp(fmt, n, k):
    g = _gen(n)
    _check_encode(torch.randn(n, k, device="cuda", generator=g).half(), fmt, 0.37 if fmt == "nv" else None)


def test_large_batches_in_a_graph_beside_a_stream():
    """Shared k, captured and replayed while another stream runs the same product: the same bits as alone."""
    g = _gen(3)
    (ac, asc, _), (wc, wsc, _) = _operand(g, "nv", 200, 8192), _operand(g, "nv", 1024, 8192)
    run = lambda: ops.gemm_fp4(ac, asc, wc, wsc, "nv")
    want = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(20):
        got.zero_()
        graph.replay()
        with torch.cuda.stream(stream):
            beside = run()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(beside, want)


def test_as_many_rows_as_there_may_be():
    """2^31 - 1 rows of 32 k by one column: the last rows, the first, and rows around 2^30."""
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB")
    m, k = 2 ** 31 - 1, 32
    a = torch.zeros(m, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full(((m + 127) // 128, 1, 512), 127, dtype=torch.uint8, device="cuda")
    rows = [0, 1, 255, 2 ** 30 - 1, 2 ** 30, m - 300, m - 257, m - 256, m - 33, m - 32, m - 2, m - 1]
    for i, r in enumerate(rows):
        a[r, 0] = 1 + i % 7  # 0.5 .. 6 in k 0
    w = torch.zeros(1, k // 2, dtype=torch.uint8, device="cuda")
    w[0, 0] = 2  # one
    out = ops.gemm_fp4(a, scales, w, ops.preprocess_fp4_scales(torch.full((1, 1), 127, dtype=torch.uint8, device="cuda")), "mx")
    for i, r in enumerate(rows):
        assert out[r].item() == ref.GRID[1 + i % 7]
        out[r] = 0
    assert out.view(torch.int16).max() == 0 and out.view(torch.int16).min() == 0
    del a, scales, out
    torch.cuda.empty_cache()
