"""Waits of the 4-bit float kernels that run out: the status says so, nothing wrong is written, and the next call is right."""
import ctypes

import pytest
import torch

from relax_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _status():
    st = ctypes.c_int(-1)
    assert _lib.load().rb200_check_async_error(None, ctypes.byref(st)) == 0
    return st.value


# every entry's 64 f are 16 or more units of k, a CTA has two or more: CTA 1 hands its first ones over
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("tokens, experts, hidden, ffn", [(1, 2, 4096, 256), (8, 2, 4096, 4096), (20, 2, 4096, 512), (32, 4, 7168, 2048)])
def test_an_expert_layer_whose_first_kernel_gave_up_writes_nothing(fmt, tokens, experts, hidden, ffn):
    lib, g, block = _lib.load(), _gen(tokens + ffn), {"mx": 32, "nv": 16}[fmt]
    byte = 120 if fmt == "mx" else 0x20
    weight = lambda n, k: (torch.randint(0, 256, (experts, n, k // 2), dtype=torch.uint8, device="cuda", generator=g),
                           ops.preprocess_fp4_scales(torch.full((experts, n, k // block), byte, dtype=torch.uint8, device="cuda")))
    (w1, s1), (w2, s2) = weight(2 * ffn, hidden), weight(hidden, ffn)
    x = (torch.randn(tokens, hidden, device="cuda", generator=g) * 0.05).half()
    logits = torch.randn(tokens, experts, device="cuda", generator=g)
    want = ops.moe_layer_fp4(x, logits, w1, s1, w2, s2, 2, fmt)
    assert torch.isfinite(want).all()
    size = ops.moe_layer_fp4_workspace_bytes(tokens, 2, hidden, ffn)
    ws = torch.full((size // 2 + 1,), 1.0, dtype=torch.float16, device="cuda")  # what h held before: ones
    out = torch.full_like(x, -7.0)
    d = _lib.MoeLayerFp4Desc()
    d.struct_size, d.format = ctypes.sizeof(_lib.MoeLayerFp4Desc), {"mx": 0, "nv": 1}[fmt]
    d.x, d.logits, d.out = x.data_ptr(), logits.data_ptr(), out.data_ptr()
    d.w_gate_up, d.gate_up_scales, d.w_down, d.down_scales = w1.data_ptr(), s1.data_ptr(), w2.data_ptr(), s2.data_ptr()
    d.tokens, d.num_experts, d.top_k, d.hidden, d.ffn = tokens, experts, 2, hidden, ffn
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    call = lambda absent: _lib.check(lib.rb200_moe_layer_fp4_selftest(ctypes.byref(d), ctypes.c_void_p(ws.data_ptr()), size, absent, stream))
    torch.cuda.synchronize()
    assert _status() == 0
    _lib.check(lib.rb200_set_wait_limit_ms(50))
    try:
        call(1)
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.rb200_set_wait_limit_ms(0))
    assert _status() == 1
    assert (out == -7.0).all()
    call(-1)
    assert torch.equal(out, want)
    assert _status() == 0


# one row block a cluster shares (quantised by the product's CTAs, and before), pairs of CTAs that share k, pairs with several tiles
@pytest.mark.parametrize("fmt, m, n, k", [("mx", 2, 4096, 4096), ("nv", 48, 4096, 4096), ("nv", 128, 1024, 8192), ("mx", 300, 22016, 2048),
                                          ("mx", 130, 520, 96)])
def test_a_product_whose_waits_run_out_writes_no_tile(fmt, m, n, k):
    """The product becomes resident beside an all-reduce that waits 4.5 s for an absent peer, and its own waits (about two seconds)
    run out behind it: tiles stay as they were (or, where a CTA came later, are right), the status says so, the next call is right."""
    lib, g = _lib.load(), _gen(m + n)
    w, ws = ops.encode_fp4(torch.randn(n, k, device="cuda", generator=g).half(), fmt)
    x = torch.randn(m, k, device="cuda", generator=g).half() / k ** 0.5
    if m <= 2:
        call = lambda **kw: ops.linear_fp4(x, w, ws, fmt, **kw)
    else:
        a, a_s = ops.encode_fp4(x, fmt)
        call = lambda **kw: ops.gemm_fp4(a, a_s, w, ws, fmt, **kw)
    right = call()
    out = torch.full((m, n), -7.0, dtype=torch.float16, device="cuda")
    assert not (right == -7.0).any()
    workspace = torch.empty(ops.linear_fp4_workspace_bytes(m, k, fmt), dtype=torch.uint8, device="cuda")
    kw = dict(workspace=workspace) if m <= 2 else {}
    nbytes = lib.rb200_allreduce_workspace_bytes(8)
    own, absent_peer = (torch.zeros(nbytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    ws2 = (ctypes.c_void_p * 2)(own.data_ptr(), absent_peer.data_ptr())
    inp, reduced = torch.randn(8, device="cuda").half(), torch.zeros(8, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    assert _status() == 0
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(lib.rb200_set_wait_limit_ms(4500))
    try:
        _lib.check(lib.rb200_allreduce_oneshot(ws2, 0, 2, ctypes.c_void_p(inp.data_ptr()), ctypes.c_void_p(reduced.data_ptr()), 8, 8, stream))
        call(out=out, **kw)
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.rb200_set_wait_limit_ms(0))
    assert _status() == 1
    assert (out == -7.0).any(), "no wait of the product ran out"
    for m0 in range(0, m, 256):
        for n0 in range(0, n, 128):
            tile = out[m0:m0 + 256, n0:n0 + 128]
            assert (tile == -7.0).all() or torch.equal(tile, right[m0:m0 + 256, n0:n0 + 128])
    assert torch.equal(call(**kw), right)
    assert _status() == 0
