"""The expert layer over weights in 4-bit floats against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import relax_b200
from relax_b200 import ops
from tests import fp4_ref as ref

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _experts(g, fmt, experts, n, k):
    """codes, tiled scales, tensor scales, float64 values [experts, n, k]; sums over k are of order one."""
    codes = torch.randint(0, 256, (experts, n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    size = 1.0 / (2.9 * np.sqrt(k))
    if fmt == "mx":
        mid = 127 + round(np.log2(size))
        scales = torch.randint(mid - 2, mid + 3, (experts, n, k // 32), dtype=torch.uint8, device="cuda", generator=g)
        ts = None
    else:
        scales = torch.randint(0x60, 0x7f, (experts, n, k // 16), dtype=torch.uint8, device="cuda", generator=g)
        ts = (0.5 + torch.rand(experts, device="cuda", generator=g)) * (size / 150)
    vals = np.stack([ref.decode(codes[e].cpu().numpy(), scales[e].cpu().numpy(), fmt, 1.0 if ts is None else float(ts[e]))
                     for e in range(experts)])
    return codes, ops.preprocess_fp4_scales(scales), ts, vals


def _layer(x, logits, top_k, renormalize, w1, w2):
    """The layer in 64 bits, and how far fp32 sums, h in fp16 and the output's rounding may take it."""
    t, experts = logits.shape
    f = w2.shape[2]
    out, err = np.zeros((t, w2.shape[1])), np.zeros((t, w2.shape[1]))
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    for i in range(t):
        order = sorted(range(experts), key=lambda e: (-logits[i, e], e))[:top_k]
        gates = p[i, order] / (p[i, order].sum() if renormalize else 1.0)
        for gate, e in zip(gates, order):
            gu = w1[e] @ x[i]
            # fp32 sums of k exact products: at most k / 16 + 32 roundings of partial sums, each below 2^-24 of the magnitudes
            d = (x.shape[1] / 16 + 32) * 2.0 ** -24 * (np.abs(w1[e]) @ np.abs(x[i]))
            gt, up = gu[:f], gu[f:]
            s = gt / (1 + np.exp(-gt))
            h = s * up
            # |silu'| <= 1.1; exp, division and two products in fp32: 2^-20; h rounds to fp16 (2^-24 apart below 2^-14)
            dh = 1.1 * d[:f] * np.abs(up) + np.abs(s) * d[f:] + d[:f] * d[f:] * 1.1 + 2.0 ** -20 * np.abs(h)
            dh += 2.0 ** -11 * (np.abs(h) + dh) + 2.0 ** -25
            out[i] += gate * (w2[e] @ h)
            # the roundings of h are independent and the sum of so many of them is held to its whole sum of magnitudes only
            # where it has few terms: six standard deviations of uniform roundings otherwise (a chance of 2e-9 per output)
            lin = np.abs(w2[e]) @ dh
            dev = 6 * np.sqrt((w2[e] ** 2) @ (dh ** 2) / 3)
            err[i] += gate * np.minimum(lin, dev + np.abs(w2[e]) @ (dh - 2.0 ** -11 * np.abs(h)).clip(0))
            err[i] += gate * (f / 16 + 32) * 2.0 ** -24 * (np.abs(w2[e]) @ np.abs(h))
            err[i] += 2.0 ** -20 * np.abs(gate * (w2[e] @ h))  # the gate's exponentials, sums and quotients
    return out, err + 2.0 ** -11 * (np.abs(out) + err) + 2.0 ** -25


def _check(got, out, err):
    got = got.double().cpu().numpy()
    bad = np.argwhere(~(np.abs(got - out) <= err))
    assert bad.size == 0, (len(bad), bad[:4], got[tuple(bad[0])], out[tuple(bad[0])], err[tuple(bad[0])])


CASES = [  # tokens, hidden, ffn, experts, top_k
    (1, 64, 64, 1, 1), (1, 128, 64, 2, 1), (1, 256, 128, 4, 2), (2, 320, 192, 3, 3), (3, 64, 1088, 8, 2), (5, 576, 64, 5, 4),
    (7, 448, 320, 33, 6), (8, 512, 512, 8, 2), (8, 192, 832, 256, 8), (9, 256, 256, 4, 2), (13, 640, 384, 16, 8), (16, 128, 128, 2, 2),
    (17, 256, 192, 3, 1), (29, 384, 448, 64, 6), (32, 256, 320, 1, 1), (32, 512, 256, 8, 8), (1, 4096, 256, 2, 2), (2, 128, 4160, 3, 2),
    # boxes of 64, 56, 48, 40 and 32 rows, whose rows lie in two scale tiles or past the matrix
    (1, 128, 8256, 2, 1), (1, 192, 6976, 2, 1), (1, 64, 5568, 3, 2), (1, 128, 3648, 4, 3), (8, 4160, 128, 3, 3), (9, 2880, 192, 4, 2),
    (4, 3584, 64, 2, 2), (20, 4096, 64, 2, 1), (1, 7168, 64, 2, 1),
]


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("tokens, hidden, ffn, experts, top_k", CASES)
def test_layer(fmt, tokens, hidden, ffn, experts, top_k):
    g = _gen(tokens * 1000 + hidden + ffn)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).half()
    logits = 2 * torch.randn(tokens, experts, device="cuda", generator=g)
    c1, s1, t1, w1 = _experts(g, fmt, experts, 2 * ffn, hidden)
    c2, s2, t2, w2 = _experts(g, fmt, experts, hidden, ffn)
    for renorm in (False, True):
        got = ops.moe_layer_fp4(x, logits, c1, s1, c2, s2, top_k, fmt, t1, t2, renormalize=renorm)
        _check(got, *_layer(x.double().cpu().numpy(), logits.double().cpu().numpy(), top_k, renorm, w1, w2))
    again = ops.moe_layer_fp4(x, logits, c1, s1, c2, s2, top_k, fmt, t1, t2, renormalize=True)
    assert torch.equal(again, got)


def _small(fmt="mx", tokens=6, experts=8, seed=1, hidden=256, ffn=192):
    g = _gen(seed)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).half()
    c1, s1, t1, w1 = _experts(g, fmt, experts, 2 * ffn, hidden)
    c2, s2, t2, w2 = _experts(g, fmt, experts, hidden, ffn)
    return g, x, (c1, s1, c2, s2), (t1, t2), (w1, w2)


def test_equal_logits_go_to_the_lower_expert():
    _, x, w, t, v = _small(tokens=4, experts=40)
    logits = torch.zeros(4, 40, device="cuda")
    logits[1, [5, 37, 36]] = 1.0
    logits[2, 39] = 3.0
    logits[3] = float("-inf")
    logits[3, 33], logits[3, 2] = -1.0, -1.0
    logits[0, 0::2] = -0.0
    got = ops.moe_layer_fp4(x, logits, *w, 3, "mx", *t)
    ref_logits = logits.double().cpu().numpy()
    _check(got, *_layer(x.double().cpu().numpy(), ref_logits, 3, False, *v))


def test_logits_that_are_not_finite_stay_with_their_token():
    g, x, w, t, _ = _small(tokens=9)
    logits = torch.randn(9, 8, device="cuda", generator=g)
    base = ops.moe_layer_fp4(x, logits, *w, 2, "mx", *t, renormalize=True)
    logits[1, 3], logits[4], logits[6, 0] = float("nan"), float("-inf"), float("inf")
    x[8, 17] = float("nan")
    for renorm in (False, True):
        out = ops.moe_layer_fp4(x, logits, *w, 2, "mx", *t, renormalize=renorm)
        assert torch.isnan(out[[1, 4, 6, 8]]).all()
    keep = [0, 2, 3, 5, 7]
    assert torch.equal(out[keep], base[keep])


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_a_token_does_not_depend_on_the_others(fmt):
    """Alone and in a batch a token takes the same products; what differs is the order of its experts' sums."""
    g, x, w, t, v = _small(fmt, tokens=31, experts=6)
    logits = torch.randn(31, 6, device="cuda", generator=g)
    out, err = _layer(x.double().cpu().numpy(), logits.double().cpu().numpy(), 2, False, *v)
    _check(ops.moe_layer_fp4(x, logits, *w, 2, fmt, *t), out, err)
    for i in (0, 13, 30):
        _check(ops.moe_layer_fp4(x[i:i + 1], logits[i:i + 1], *w, 2, fmt, *t), out[i:i + 1], err[i:i + 1])


def test_all_tokens_to_one_expert_and_unused_nan_experts():
    g, x, w, t, v = _small(tokens=32, experts=4)
    logits = torch.full((32, 4), -5.0, device="cuda")
    logits[:, 2] = 5.0
    for e in (0, 1, 3):  # weights that no token needs must not be seen
        w[1][e] = 255
        w[3][e] = 255
    got = ops.moe_layer_fp4(x, logits, *w, 1, "mx", *t)
    _check(got, *_layer(x.double().cpu().numpy(), logits.double().cpu().numpy(), 1, False, *v))


def test_strides_types_outputs_and_empty_batches():
    g, x, w, t, _ = _small(tokens=5)
    logits = torch.randn(5, 8, device="cuda", generator=g)
    want = ops.moe_layer_fp4(x, logits, *w, 2, "mx")
    wide = torch.zeros(5, 300, device="cuda").half()
    wide[:, 3:259] = x
    assert torch.equal(ops.moe_layer_fp4(wide[:, 3:259], logits.double(), *w, 2, "mx"), want)
    ws = torch.empty(ops.moe_layer_fp4_workspace_bytes(5, 2, 256, 192), dtype=torch.uint8, device="cuda")
    out = torch.zeros(6, 256, device="cuda").half()
    assert torch.equal(ops.moe_layer_fp4(x, logits, *w, 2, "mx", workspace=ws, out=out[:5]), want)
    assert not out[5].any()
    assert ops.moe_layer_fp4(x[:0], logits[:0], *w, 2, "mx").shape == (0, 256)


def test_refusals_of_shapes():
    g, x, w, t, _ = _small(tokens=5)
    logits = torch.randn(5, 8, device="cuda", generator=g)
    with pytest.raises(relax_b200.RB200Error, match="logits"):
        ops.moe_layer_fp4(x, logits[:4], *w, 2, "mx")
    with pytest.raises(relax_b200.RB200Error, match="tokens=33"):
        ops.moe_layer_fp4(x[:1].expand(33, 256), logits[:1].expand(33, 8), *w, 2, "mx")
    with pytest.raises(relax_b200.RB200Error, match="scales"):
        ops.moe_layer_fp4(x, logits, *w, 2, "nv")
    with pytest.raises(relax_b200.RB200Error, match="w_gate_up"):
        ops.moe_layer_fp4(x, logits, w[0][:, :-64], w[1], w[2], w[3], 2, "mx")
    with pytest.raises(relax_b200.RB200Error, match="dtype"):
        ops.moe_layer_fp4(x.float(), logits, *w, 2, "mx")


def test_beside_the_grouped_matmuls():
    """The routing agrees with moe_route, so the layer is route, gather, two products per expert and combine."""
    g, x, w, t, v = _small("nv", tokens=12, experts=16)
    logits = torch.randn(12, 16, device="cuda", generator=g)
    indptr, tok, gate, rof = ops.moe_route(logits, 4)
    xg = ops.moe_gather(x, tok)
    y = torch.zeros(48, 256, device="cuda").half()
    begin = 0
    for e, end in enumerate(indptr.tolist()):
        if end > begin:
            gu = torch.from_numpy(v[0][e]).cuda() @ xg[begin:end].double().T
            h = (torch.nn.functional.silu(gu[:192]) * gu[192:]).half().double()
            y[begin:end] = (torch.from_numpy(v[1][e]).cuda() @ h).T.half()
        begin = end
    want = ops.moe_combine(y, rof, gate, 4)
    got = ops.moe_layer_fp4(x, logits, *w, 4, "nv", *t)
    assert (got.float() - want.float()).abs().max() <= 4e-3 * want.float().abs().max()


def test_layers_in_a_graph_and_on_streams():
    layers = []
    for i in range(3):
        g, x, w, t, _ = _small("mx", tokens=7, seed=i)
        layers.append((torch.randn(7, 8, device="cuda", generator=g), w))

    def chain(y):
        # (a layer about squares its input's size: without the scaling the third one's h, as fp32 sums too, is beyond fp16)
        for logits, w in layers:
            y = ops.moe_layer_fp4(y, logits, *w, 2, "mx", renormalize=True) * 0.125
        return y

    want = chain(x)
    assert torch.isfinite(want).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [chain(x) for _ in range(20)]
    here = [chain(x) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got + here)
    buf, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(buf)
    for i in range(20):
        buf.copy_(x if i % 2 else -x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, chain(x if i % 2 else -x))


def test_logits_written_by_the_kernel_before():
    """New logits and activations for every call, back to back."""
    g, x, w, t, _ = _small(tokens=8)
    all_logits = torch.randn(30, 8, 8, device="cuda", generator=g)
    logits, y = torch.empty(8, 8, device="cuda"), torch.empty_like(x)
    got = []
    for l in all_logits:
        logits.copy_(l)
        y.copy_(x * l[0, 0])
        got.append(ops.moe_layer_fp4(y, logits, *w, 2, "mx"))
    for l, o in zip(all_logits, got):
        torch.cuda.synchronize()
        assert torch.equal(ops.moe_layer_fp4((x * l[0, 0]).contiguous(), l.contiguous(), *w, 2, "mx"), o)
