"""Linears over 4-bit floats: results over their own inputs, batches around the rules that choose a kernel, odd values."""
import ctypes

import numpy as np
import pytest
import torch

import relax_b200
from relax_b200 import _lib, ops
from tests import fp4_ref as ref
from tests.test_fp4_gpu import TYPES, _check_product, _gen, _np, _operand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m, n", [(1, 512), (2, 4096), (4, 288), (20, 512), (64, 288), (70, 512), (300, 512)])
def test_result_over_the_activations(fmt, dtype, m, n):
    """Tiles of a small batch store while others still need all of x: with out = x it has to be quantised first."""
    g = _gen(m + n)
    (wc, wsc, _) = _operand(g, fmt, n, n)
    ts = torch.tensor([2.0 ** -10], device="cuda") if fmt == "nv" else None
    x = (torch.randn(m, n, device="cuda", generator=g)).to(TYPES[dtype])
    call = lambda v, **kw: ops.linear_fp4(v, wc, wsc, fmt, x_tensor_scale=ts, w_tensor_scale=ts, **kw)
    want, with_x = call(x), call(x, residual=x, binary_op="plus")
    for _ in range(5):
        y = x.clone()
        assert call(y, out=y) is y and torch.equal(y, want)
        y = x.clone()
        assert torch.equal(call(y, residual=y, binary_op="plus", out=y), with_x)


def test_result_over_a_part_of_the_activations():
    """The last row of x is the first of out."""
    g, k = _gen(1), 256
    wc, wsc, _ = _operand(g, "mx", k, k)
    base = torch.randn(3, k, device="cuda", generator=g).half()
    want = ops.linear_fp4(base[:2].clone(), wc, wsc, "mx")
    assert torch.equal(ops.linear_fp4(base[:2], wc, wsc, "mx", out=base[1:]), want)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m", [1, 3, 40, 80, 300])
@pytest.mark.parametrize("act, un", [("relu", "identity"), ("identity", "relu"), ("silu", "relu")])
def test_a_bad_block_is_seen_through_relu(fmt, dtype, m, act, un):
    """A row of x, a row of w and an element of bias that are not finite: their outputs are NaN, the others as without."""
    g, n, k = _gen(m), 200, 320
    x = torch.randn(m, k, device="cuda", generator=g).to(TYPES[dtype])
    w = torch.randn(n, k, device="cuda", generator=g).to(TYPES[dtype])
    bias = torch.randn(n, device="cuda", generator=g).to(TYPES[dtype])

    def call(x, w, bias):
        wc, wsc = ops.encode_fp4(w, fmt)
        return ops.linear_fp4(x, wc, wsc, fmt, bias=bias, activation=act, unary_op=un)

    base = call(x, w, bias)
    assert (base >= 0).all()
    y, v, b = x.clone(), w.clone(), bias.clone()
    y[m // 2, 100], v[150, 5], b[7] = float("inf"), float("nan"), float("nan")
    got = call(y, v, b)
    assert torch.isnan(got[m // 2]).all() and torch.isnan(got[:, [7, 150]]).all()
    got[m // 2], got[:, [7, 150]] = base[m // 2], base[:, [7, 150]]
    assert torch.equal(got, base)


def test_a_residual_or_a_result_of_another_shape_is_refused():
    """As many elements in another order are not the same matrix."""
    g, m, n, k = _gen(2), 6, 96, 64
    wc, wsc, _ = _operand(g, "mx", n, k)
    x = torch.randn(m, k, device="cuda", generator=g).half()
    r = torch.randn(m, n, device="cuda", generator=g).half()
    ac, asc = ops.encode_fp4(x, "mx")
    calls = [lambda **kw: ops.linear_fp4(x, wc, wsc, "mx", binary_op="plus", **kw),
             lambda **kw: ops.gemm_fp4(ac, asc, wc, wsc, "mx", binary_op="plus", **kw)]
    for call in calls:
        want = call(residual=r)
        assert torch.equal(call(residual=r.view(1, m, n)), want)
        for bad in (r.view(n, m), r.view(-1), r.view(m, n // 2, 2)):
            with pytest.raises(relax_b200.RB200Error, match="residual must be"):
                call(residual=bad)
    decode = relax_b200.get_global_func("relax_b200.decode_fp4")
    with pytest.raises(relax_b200.RB200Error, match="out must be"):
        decode(ac, asc, "mx", None, torch.empty(k, m, dtype=torch.float16, device="cuda"))
    assert ops.linear_fp4(x[0], wc, wsc, "mx", residual=r[0], binary_op="plus").shape == (n,)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_no_rows_with_everything_a_call_can_have(fmt):
    g, n, k = _gen(6), 96, 64
    wc, wsc, _ = _operand(g, fmt, n, k)
    x, r, b = torch.empty(0, k, device="cuda").half(), torch.empty(0, n, device="cuda").half(), torch.zeros(n, device="cuda").half()
    ts = torch.ones(1, device="cuda") if fmt == "nv" else None
    kw = dict(bias=b, residual=r, activation="silu", binary_op="plus", unary_op="relu")
    assert ops.linear_fp4(x, wc, wsc, fmt, ts, ts, **kw).shape == (0, n)
    assert ops.linear_fp4(x.view(0, 3, k), wc, wsc, fmt, ts, ts, **{**kw, "residual": r.view(0, 3, n)}).shape == (0, 3, n)
    ac, asc = ops.encode_fp4(x, fmt, tensor_scale=ts)
    assert ops.gemm_fp4(ac, asc, wc, wsc, fmt, ts, ts, **kw).shape == (0, n)
    assert ops.decode_fp4(ac, asc, fmt, tensor_scale=ts).shape == (0, k)


# Batches quantised by the product's CTAs: one and two rows; three and four with at most four chunks of 256 k a CTA (a cluster shares
# k 8192 and k 10240 by eight, k 1024 and k 1280 are one CTA's at 19000 columns).  Next to each its neighbour that is not.
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m, n, k", [(1, 130, 32), (1, 300, 992), (2, 200, 288), (2, 129, 4128), (3, 130, 288), (3, 300, 992), (4, 130, 288),
                                     (4, 129, 992), (5, 129, 992), (4, 136, 8192), (4, 136, 8224), (4, 130, 10240), (3, 19000, 1024),
                                     (4, 19000, 1024), (4, 19000, 1280), (5, 19000, 1024)])
def test_few_rows(fmt, dtype, m, n, k):
    g = _gen(m * n + k)
    x = (torch.randn(m, k, device="cuda", generator=g) * torch.exp(torch.randn(k, device="cuda", generator=g))).to(TYPES[dtype])
    x[m - 1, k // 2:] *= 2.0 ** -6  # rows of other scales
    wc, wsc, w = _operand(g, fmt, n, k)
    ts = (x.abs().amax().float() / 2688).reshape(1) if fmt == "nv" else None
    tsv = 1.0 if ts is None else float(ts)
    out = ops.linear_fp4(x, wc, wsc, fmt, x_tensor_scale=ts)
    codes, scales = ref.encode(_np(x), fmt, tsv)
    _check_product(out, ref.decode(codes, scales, fmt), w, tsv)
    ac, asc = ops.encode_fp4(x, fmt, tensor_scale=ts)
    assert torch.equal(ops.gemm_fp4(ac, asc, wc, wsc, fmt, a_tensor_scale=ts, dtype=x.dtype), out)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m", [1, 2, 3, 4])
def test_few_rows_that_are_not_finite(fmt, m):
    """A bad block of one row, in the product that quantises: NaN in that row, the others as without."""
    g, n, k = _gen(m), 200, 288
    x = torch.randn(m, k, device="cuda", generator=g).half()
    wc, wsc, _ = _operand(g, fmt, n, k)
    base = ops.linear_fp4(x, wc, wsc, fmt)
    x[m - 1, k - 1] = float("-inf")
    got = ops.linear_fp4(x, wc, wsc, fmt)
    assert torch.isnan(got[m - 1]).all() and torch.equal(got[:m - 1], base[:m - 1])


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_a_weight_quantised_by_the_call_before(fmt, m):
    """With launch overlap off: codes and scales written over and over into the same memory, each used by the next call."""
    assert not relax_b200.get_launch_overlap()
    g, n, k, times = _gen(m), 520, 1056, 30
    x = torch.randn(m, k, device="cuda", generator=g).half()
    weights = [torch.randn(n, k, device="cuda", generator=g).half() for _ in range(times)]
    codes, scales = ops.encode_fp4(weights[0], fmt)
    encode = relax_b200.get_global_func("relax_b200.encode_fp4")
    got = []
    for w in weights:
        encode(w, fmt, None, codes, scales)
        got.append(ops.linear_fp4(x, codes, scales, fmt))
    for w, y in zip(weights, got):
        c, s = ops.encode_fp4(w, fmt)
        torch.cuda.synchronize()
        assert torch.equal(ops.linear_fp4(x, c, s, fmt), y)
