"""Expert layers over 4-bit floats whose values between the two products lie far outside fp16's range."""
import numpy as np
import pytest
import torch

from relax_b200 import ops
from tests import fp4_ref as ref
from tests.test_fp4_moe_gpu import _check, _gen

pytestmark = pytest.mark.gpu


def _weights(g, fmt, experts, n, k, size):
    """codes, tiled scales, tensor scales, float64 values; sums over k of numbers of order one are about `size`."""
    codes = torch.randint(0, 256, (experts, n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    unit = size / (2.9 * np.sqrt(k))
    if fmt == "mx":
        mid = 127 + round(np.log2(unit))
        scales, ts = torch.randint(mid - 1, mid + 2, (experts, n, k // 32), dtype=torch.uint8, device="cuda", generator=g), None
    else:
        scales = torch.randint(0x60, 0x7f, (experts, n, k // 16), dtype=torch.uint8, device="cuda", generator=g)
        ts = (0.5 + torch.rand(experts, device="cuda", generator=g)) * (unit / 150)
    vals = np.stack([ref.decode(codes[e].cpu().numpy(), scales[e].cpu().numpy(), fmt, 1.0 if ts is None else float(ts[e]))
                     for e in range(experts)])
    return codes, ops.preprocess_fp4_scales(scales), ts, vals


def _layer(x, logits, top_k, w1, w2):
    """In 64 bits, and how far it may be off: the sums and functions of fp32, h as it is held, the output's rounding."""
    tokens, experts = logits.shape
    f = w2.shape[2]
    out, err = np.zeros((tokens, w2.shape[1])), np.zeros((tokens, w2.shape[1]))
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    for i in range(tokens):
        for e in sorted(range(experts), key=lambda e: (-logits[i, e], e))[:top_k]:
            gu = w1[e] @ x[i]
            # at most k / 16 + 32 roundings of partial sums, each below 2^-24 of the magnitudes, and the tensor scale's product
            d = (x.shape[1] / 16 + 33) * 2.0 ** -24 * (np.abs(w1[e]) @ np.abs(x[i]))
            gt, up = gu[:f], gu[f:]
            s = gt / (1 + np.exp(-np.clip(gt, -700, 700)))
            h = s * up
            # |silu'| <= 1.1; silu in fp32 2^-20 of its input (1 / (1 + exp) below 2^-126 is 0); a product
            dh = 1.1 * (d[:f] + 2.0 ** -20 * np.abs(gt)) * (np.abs(up) + d[f:]) + np.abs(s) * d[f:] + 2.0 ** -23 * np.abs(h)
            # 11 bits: 2^-12 of itself; fp16's last place is worth 2^-24, rounded to 2^-25, under the power of two of its sixteen and
            # once more under the row's: 2^-4 in the ordinary range, else at most twice the largest (which becomes 2^-1 to 2^15)
            top = (np.abs(h) + dh).max()
            dh += 2.0 ** -12 * (np.abs(h) + dh) + 2 * 2.0 ** -25 * (2.0 ** -4 if 2.0 ** -16 <= top < 2.0 ** 11 else 2 * top)
            y = w2[e] @ h
            out[i] += p[i, e] * y
            err[i] += p[i, e] * (np.abs(w2[e]) @ dh + (f / 16 + 33) * 2.0 ** -24 * (np.abs(w2[e]) @ (np.abs(h) + dh)) + 2.0 ** -20 * np.abs(y))
    return out, err + 2.0 ** -11 * (np.abs(out) + err) + 2.0 ** -25


# tokens, hidden, ffn, experts, top_k: entries of eight rows, of sixteen, of several
SHAPES = [(1, 256, 64, 1, 1), (3, 320, 1088, 3, 2), (9, 256, 192, 4, 2), (29, 192, 640, 3, 2), (8, 512, 320, 2, 2)]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("tokens, hidden, ffn, experts, top_k", SHAPES)
@pytest.mark.parametrize("size", [2.0 ** 6, 320.0, 2.0 ** 40, 2.0 ** -9, 2.0 ** -12, 2.0 ** -30])
def test_sizes_of_h(fmt, tokens, hidden, ffn, experts, top_k, size):
    """gate and up of about `size` (below one, gate * up is about half its square), outputs of order one."""
    g = _gen(tokens + ffn)
    h = size * size if size > 1 else size * size / 2
    x = torch.randn(tokens, hidden, device="cuda", generator=g).half()
    logits = torch.randn(tokens, experts, device="cuda", generator=g)
    c1, s1, t1, w1 = _weights(g, fmt, experts, 2 * ffn, hidden, size)
    c2, s2, t2, w2 = _weights(g, fmt, experts, hidden, ffn, 1.0 / h)
    got = ops.moe_layer_fp4(x, logits, c1, s1, c2, s2, top_k, fmt, t1, t2)
    want, err = _layer(x.double().cpu().numpy(), logits.double().cpu().numpy(), top_k, w1, w2)
    assert 0.01 < np.abs(want).max() < 1000
    _check(got, want, err)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_sizes_within_a_row(fmt):
    """Sixteens of f that are far apart: the small ones next to large ones, alone in their row, and zeros."""
    g, experts, hidden, ffn = _gen(4), 2, 256, 320
    x = torch.randn(7, hidden, device="cuda", generator=g).half()
    x[5] = 0
    logits = torch.randn(7, experts, device="cuda", generator=g)
    c1, s1, t1, w1 = _weights(g, fmt, experts, 2 * ffn, hidden, 2.0 ** 8)
    # up rows 48 to 159 see k 0 and 1 alone, where x is small; 160 to 223 see nothing
    up = c1[:, ffn:].clone()
    up[:, 48:160, 1:] = 0
    up[:, 160:224] = 0
    c1[:, ffn:] = up
    w1 = w1.copy()
    w1[:, ffn + 48:ffn + 160, 2:] = 0
    w1[:, ffn + 160:ffn + 224] = 0
    x[:, :2] *= 2.0 ** -12
    c2, s2, t2, w2 = _weights(g, fmt, experts, hidden, ffn, 2.0 ** -14)
    got = ops.moe_layer_fp4(x, logits, c1, s1, c2, s2, 2, fmt, t1, t2)
    _check(got, *_layer(x.double().cpu().numpy(), logits.double().cpu().numpy(), 2, w1, w2))
    assert not got[5].any()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("tokens", [8, 30])
def test_a_token_beside_a_large_one(fmt, tokens):
    """A token keeps its bits whatever range the others' values need; an infinite one stays with itself."""
    g, experts, hidden, ffn = _gen(tokens), 2, 320, 448
    x = torch.randn(tokens, hidden, device="cuda", generator=g).half()
    logits = torch.randn(tokens, experts, device="cuda", generator=g)
    c1, s1, t1, _ = _weights(g, fmt, experts, 2 * ffn, hidden, 4.0)
    c2, s2, t2, _ = _weights(g, fmt, experts, hidden, ffn, 2.0 ** -8)
    call = lambda v: ops.moe_layer_fp4(v, logits, c1, s1, c2, s2, 2, fmt, t1, t2)
    want = call(x)
    assert torch.isfinite(want).all()
    y = x.clone()
    y[1] *= 2.0 ** 6
    y[2] *= 2.0 ** -14
    y[4, 7] = float("inf")
    y[6] = 0
    got = call(y)
    assert torch.isfinite(got[[1, 2]]).all() and got[1].abs().max() > 10 and not torch.isfinite(got[4]).any() and not got[6].any()
    for i in (0, 3, 5, 7):
        assert torch.equal(got[i], want[i])


def test_large_values_in_a_graph_and_on_a_stream():
    g = _gen(2)
    x = torch.randn(5, 256, device="cuda", generator=g).half()
    logits = torch.randn(5, 4, device="cuda", generator=g)
    c1, s1, _, _ = _weights(g, "mx", 4, 2 * 576, 256, 2.0 ** 10)
    c2, s2, _, _ = _weights(g, "mx", 4, 256, 576, 2.0 ** -20)
    call = lambda v: ops.moe_layer_fp4(v, logits, c1, s1, c2, s2, 2, "mx")
    # two sizes in turn: the words and exponents of one call mean nothing to the next
    small = (x * 2.0 ** -9).half()
    want, want_small = call(x), call(small)
    assert torch.isfinite(want).all() and want.abs().max() > 0.1
    buf, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(buf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(20):
        buf.copy_(small if i % 2 else x)
        graph.replay()
        with torch.cuda.stream(side):
            beside = call(x if i % 2 else small)
        torch.cuda.synchronize()
        assert torch.equal(out, want_small if i % 2 else want) and torch.equal(beside, want if i % 2 else want_small)
