"""The 4-bit float operators as a program uses them: together, on streams, in graphs, through the C ABI and the registry."""
import ctypes

import pytest
import torch

import relax_b200
from relax_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weight(g, fmt, n, k, experts=None):
    shape = (n, k) if experts is None else (experts, n, k)
    w = torch.randn(shape, device="cuda", generator=g) / k ** 0.5
    ts = None
    if fmt == "nv":
        ts = (w.abs().amax(dim=(-2, -1)) / 2688).reshape(-1)
    return ops.encode_fp4(w.half(), fmt, tensor_scale=ts) + (ts,)


class Layer:
    """An attention-less decoder layer: two linears with a residual, then an expert layer."""

    def __init__(self, g, fmt, hidden=512, ffn=256, experts=8):
        self.fmt = fmt
        self.a, self.b = _weight(g, fmt, hidden, hidden), _weight(g, fmt, hidden, hidden)
        self.up, self.down = _weight(g, fmt, 2 * ffn, hidden, experts), _weight(g, fmt, hidden, ffn, experts)
        self.router = torch.randn(experts, hidden, device="cuda", generator=g) / hidden ** 0.5
        self.xts = torch.tensor([6.0 / 2688], device="cuda") if fmt == "nv" else None

    def __call__(self, x):
        y = ops.linear_fp4(x, self.a[0], self.a[1], self.fmt, self.xts, self.a[2], activation="silu")
        x = ops.linear_fp4(y, self.b[0], self.b[1], self.fmt, self.xts, self.b[2], residual=x, binary_op="plus")
        x = x / x.float().pow(2).mean(-1, keepdim=True).sqrt().half()
        logits = x.float() @ self.router.T
        if x.shape[0] <= 32:
            return x + ops.moe_layer_fp4(x, logits, self.up[0], self.up[1], self.down[0], self.down[1], 2, self.fmt, self.up[2],
                                         self.down[2], renormalize=True)
        return x


def _plain(layer, x):
    """The same with the weights read back and the activations quantised and read back, in 64 bits."""
    fmt = layer.fmt

    def back(w):
        return ops.decode_fp4(w[0], w[1], fmt, tensor_scale=w[2], dtype=torch.float32).double()

    def act(v):
        c, s = ops.encode_fp4(v, fmt, tensor_scale=layer.xts)
        return ops.decode_fp4(c, s, fmt, tensor_scale=layer.xts, dtype=torch.float32).double()

    y = torch.nn.functional.silu(act(x) @ back(layer.a).T).half()
    x = (act(y) @ back(layer.b).T + x.double()).half()
    x = x / x.float().pow(2).mean(-1, keepdim=True).sqrt().half()
    if x.shape[0] > 32:
        return x.double()
    p = torch.softmax((x.float() @ layer.router.T).double(), -1)
    top, idx = p.topk(2, -1)
    top = top / top.sum(-1, keepdim=True)
    up, down, out = back(layer.up), back(layer.down), x.double().clone()
    for t in range(x.shape[0]):
        for j in range(2):
            gu = up[idx[t, j]] @ x[t].double()
            f = gu.shape[0] // 2
            out[t] += top[t, j] * (down[idx[t, j]] @ (torch.nn.functional.silu(gu[:f]) * gu[f:]))
    return out


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("tokens", [1, 6, 29, 100])
def test_layers_together(fmt, tokens):
    g = _gen(tokens)
    layers = [Layer(g, fmt) for _ in range(2)]
    x = torch.randn(tokens, 512, device="cuda", generator=g).half()
    y = x
    for layer in layers:
        want = _plain(layer, y)
        y = layer(y)
        # a code of an activation in between may fall to the other side of its border (a sixth of its block's largest value, in one
        # of 512 products of 1/sqrt(512)): a percent of the outputs' scale; else roundings to fp16
        assert (y.double() - want).abs().max() <= 0.03 * want.abs().max()
        assert (y.double() - want).norm() <= 3e-3 * want.norm()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("tokens", [2, 11, 70])
def test_layers_in_graphs_and_on_two_streams(fmt, overlap, tokens):
    g = _gen(3)
    layers = [Layer(g, fmt) for _ in range(2)]
    x = torch.randn(tokens, 512, device="cuda", generator=g).half()

    def run(v):
        for layer in layers:
            v = layer(v)
        return v

    want, other = run(x), run(-x)
    torch.cuda.synchronize()
    before = relax_b200.get_launch_overlap()
    relax_b200.set_launch_overlap(overlap)
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = []
        for _ in range(10):
            with torch.cuda.stream(side):
                got.append(run(x))
            assert torch.equal(run(-x), other)
        torch.cuda.synchronize()
        assert all(torch.equal(v, want) for v in got)
        buf, graphs = x.clone(), []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = run(buf)
            graphs.append((graph, out))
    finally:
        relax_b200.set_launch_overlap(before)
    for i in range(10):
        buf.copy_(x if i % 2 else -x)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want if i % 2 else other)


def test_expert_layers_without_hand_over_words():
    """There are 32 areas of them; graphs keep theirs, so the last ones here have none and compute whole tiles."""
    g = _gen(5)
    layer = Layer(g, "mx", hidden=512, ffn=1088)
    x = torch.randn(3, 512, device="cuda", generator=g).half()
    logits = x.float() @ layer.router.T
    call = lambda: ops.moe_layer_fp4(x, logits, layer.up[0], layer.up[1], layer.down[0], layer.down[1], 2, "mx")
    want = call()
    graphs = []
    for _ in range(36):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for graph, out in graphs:
        out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for graph, out in graphs:  # another order of sums: a rounding of h (2^-11) and of the output
        assert (out.float() - want.float()).abs().max() <= 2.0 ** -9 * want.float().abs().max()
    del graphs


def _check(rc):
    _lib.check(rc)


@pytest.mark.parametrize("m", [1, 20, 64, 65, 300])
@pytest.mark.parametrize("dtype, code", [(torch.float16, 0), (torch.bfloat16, 1), (torch.float32, 2)])
def test_row_strides_through_the_c_abi(m, dtype, code):
    """Rows of a wider x and of a wider out; what lies between and behind the rows stays as it was."""
    lib, n, k = _lib.load(), 200, 288
    g = _gen(m)
    w, ws, _ = _weight(g, "mx", n, k)
    x = torch.randn(m + 1, k + 32, device="cuda", generator=g).to(dtype)
    out = torch.full((m + 2, n + 24), 7.0, device="cuda").to(dtype)
    bias = torch.randn(n, device="cuda", generator=g).to(dtype)
    d = _lib.GemmFp4Desc()
    d.struct_size, d.format, d.out_dtype = ctypes.sizeof(_lib.GemmFp4Desc), 0, code
    d.w, d.w_scales, d.bias, d.out = w.data_ptr(), ws.data_ptr(), bias.data_ptr(), out.data_ptr()
    d.m, d.n, d.k, d.ldo = m, n, k, n + 24
    size = lib.rb200_linear_fp4_workspace_bytes(m, k, 0)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _check(lib.rb200_linear_fp4(ctypes.c_void_p(x.data_ptr()), code, k + 32, ctypes.byref(d), ctypes.c_void_p(space.data_ptr()), size, stream))
    torch.cuda.synchronize()
    want = ops.linear_fp4(x[:m, :k].contiguous(), w, ws, "mx", bias=bias)
    assert torch.equal(out[:m, :n], want)
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("m", [3, 40, 200])
def test_residual_in_place(m):
    g = _gen(m)
    w, ws, _ = _weight(g, "mx", 264, 512)
    x = torch.randn(m, 512, device="cuda", generator=g).half()
    r = torch.randn(m, 264, device="cuda", generator=g).half()
    want = ops.linear_fp4(x, w, ws, "mx", residual=r, binary_op="plus")
    assert ops.linear_fp4(x, w, ws, "mx", residual=r, binary_op="plus", out=r) is r
    assert torch.equal(r, want)


def test_expert_layer_in_place():
    g = _gen(9)
    layer = Layer(g, "nv")
    x = torch.randn(7, 512, device="cuda", generator=g).half()
    logits = x.float() @ layer.router.T
    args = (logits, layer.up[0], layer.up[1], layer.down[0], layer.down[1], 2, "nv", layer.up[2], layer.down[2])
    want = ops.moe_layer_fp4(x, *args)
    assert torch.equal(ops.moe_layer_fp4(x, *args, out=x), want) and torch.equal(x, want)


def test_through_the_registry():
    g = _gen(11)
    w, ws, _ = _weight(g, "mx", 96, 128)
    x = torch.randn(5, 128, device="cuda", generator=g).half()
    f = relax_b200.get_global_func
    codes = torch.empty(5, 64, dtype=torch.uint8, device="cuda")
    scales = torch.empty(1, 1, 512, dtype=torch.uint8, device="cuda")
    f("relax_b200.encode_fp4")(x, "mx", None, codes, scales)
    out = torch.empty(5, 96, dtype=torch.float16, device="cuda")
    f("relax_b200.gemm_fp4")(codes, scales, w, ws, "mx", None, None, None, None, "", "", "", out)
    assert torch.equal(out, ops.linear_fp4(x, w, ws, "mx"))
    bound = f("relax_b200.decode_fp4").bind(codes, scales, "mx", None, x)
    bound()
    assert torch.equal(x, ops.decode_fp4(codes, scales, "mx"))
    with pytest.raises(relax_b200.RB200Error, match="expected"):
        f("relax_b200.gemm_fp4")(codes, scales[:, :, :256].contiguous(), w, ws, "mx", None, None, None, None, "", "", "", out)
    with pytest.raises(relax_b200.RB200Error, match="k="):
        f("relax_b200.gemm_fp4")(codes[:, :32].contiguous(), scales, w, ws, "mx", None, None, None, None, "", "", "", out)
    with pytest.raises(relax_b200.RB200Error, match="bias"):
        ops.linear_fp4(x, w, ws, "mx", bias=torch.zeros(96, device="cuda"))
    with pytest.raises(relax_b200.RB200Error, match="tensor scale"):
        ops.linear_fp4(x, w, ws, "mx", w_tensor_scale=torch.ones(1, device="cuda"))
    with pytest.raises(relax_b200.RB200Error, match="workspace"):
        ops.linear_fp4(x, w, ws, "mx", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_no_wait_ran_out():
    torch.cuda.synchronize()
    st = ctypes.c_int(-1)
    assert _lib.load().rb200_check_async_error(None, ctypes.byref(st)) == 0 and st.value == 0
