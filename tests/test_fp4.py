"""Microscaled 4-bit floats without a GPU: the reference's own consistency, and what the entry points refuse."""
import ctypes

import numpy as np
import pytest
import torch

import relax_b200
from relax_b200 import _lib, ops
from tests import fp4_ref as ref


def test_reference_round_trip():
    codes = np.arange(256, dtype=np.uint8).reshape(2, 128)[:, :64]
    for fmt, byte in (("mx", 127), ("nv", 0x38)):
        scales = np.full((2, 128 // ref.BLOCK[fmt]), byte, dtype=np.uint8)
        x = ref.decode(codes, scales, fmt)
        assert np.abs(x).max() == 6.0
        c, s = ref.encode(x, fmt)
        assert np.array_equal(ref.decode(c, s, fmt), x)


def test_reference_ties_go_to_the_even_code():
    mag = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, 7.9])
    assert ref.codes_of(mag).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7]
    # e4m3 1.0625 lies between 1.0 (even) and 1.125, 1.1875 between 1.125 and 1.25 (even)
    x = np.zeros((2, 16))
    x[0, 0], x[1, 0] = 6 * 1.0625, 6 * 1.1875
    assert ref.encode(x, "nv")[1].ravel().tolist() == [0x38, 0x3a]


def test_scale_bytes():
    lib = _lib.load()
    for rows, k, blocks, fmt in [(1, 32, 1, 0), (128, 128, 4, 0), (129, 160, 5, 0), (128, 160, 10, 1)]:
        assert lib.rb200_fp4_scale_bytes(rows, k, fmt) == (rows + 127) // 128 * ((blocks + 3) // 4) * 512
    assert lib.rb200_fp4_scale_bytes(1, 32, 2) == 0


def test_global_names():
    names = relax_b200.list_global_func_names()
    for n in ("encode_fp4", "decode_fp4", "preprocess_fp4_scales", "gemm_fp4", "linear_fp4"):
        assert "relax_b200." + n in names


def _error(rc):
    assert rc == -1
    return _lib.load().rb200_last_error().decode()


def test_encode_refusals():
    lib, p = _lib.load(), ctypes.c_void_p(256)
    enc = lambda x=p, dt=0, batch=1, rows=4, k=64, ldx=64, fmt=0, ts=None, c=p, s=p: lib.rb200_encode_fp4(
        x, dt, batch, rows, k, ldx, fmt, ts, c, s, None)
    assert "format" in _error(enc(fmt=2))
    assert "k % 32" in _error(enc(k=48))
    assert "k % 32" in _error(enc(k=0))
    assert "element type" in _error(enc(dt=3))
    assert "non-NULL" in _error(enc(x=None))
    assert "tensor scale" in _error(enc(ts=p))
    assert "aligned" in _error(enc(ldx=60))
    assert "aligned" in _error(enc(ldx=68))
    assert "aligned" in _error(enc(x=ctypes.c_void_p(258)))
    assert "aligned" in _error(enc(c=ctypes.c_void_p(264)))
    assert "batch" in _error(enc(batch=-1))
    assert enc(rows=0) == 0 and enc(batch=0) == 0
    assert "element type" in _error(lib.rb200_decode_fp4(p, p, 1, 4, 64, 0, None, p, 5, None))
    assert "non-NULL" in _error(lib.rb200_decode_fp4(p, p, 1, 4, 64, 0, None, None, 0, None))
    assert "different" in _error(lib.rb200_preprocess_fp4_scales(p, p, 1, 4, 64, 0, None))


def _desc(**kw):
    d = _lib.GemmFp4Desc()
    d.struct_size = ctypes.sizeof(_lib.GemmFp4Desc)
    for name in ("a", "a_scales", "w", "w_scales", "out"):
        setattr(d, name, 256)
    d.m, d.n, d.k, d.ldo = 4, 16, 64, 16
    for name, v in kw.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("change, words", [
    (dict(struct_size=8), "struct_size"), (dict(format=3), "format"), (dict(k=100), "k % 32"), (dict(n=0), "n=0"),
    (dict(out_dtype=7), "element type"), (dict(activation=4), "activation"), (dict(activation=-1), "activation"),
    (dict(binary_op=3, residual=256), "binary op"), (dict(unary_op=2), "unary op"), (dict(binary_op=1), "residual"),
    (dict(residual=256), "residual"), (dict(ldo=8), "ldo"), (dict(a_tensor_scale=256), "tensor scale"),
    (dict(w_tensor_scale=256), "tensor scale"), (dict(w=None), "non-NULL"), (dict(out=None), "non-NULL"),
    (dict(w=264), "aligned"), (dict(out=257), "aligned"), (dict(bias=257), "aligned"), (dict(a=None), "a and a_scales"),
    (dict(a_scales=264), "a and a_scales"), (dict(m=-1), "rows"),
])
def test_gemm_refusals(change, words):
    lib = _lib.load()
    assert words in _error(lib.rb200_gemm_fp4(ctypes.byref(_desc(**change)), None))


def test_linear_refusals():
    lib, p = _lib.load(), ctypes.c_void_p(256)
    need = lib.rb200_linear_fp4_workspace_bytes(4, 64, 0)
    lin = lambda x=p, dt=0, ldx=64, ws=p, size=need, **kw: lib.rb200_linear_fp4(x, dt, ldx, ctypes.byref(_desc(**kw)), ws, size, None)
    assert "element type" in _error(lin(dt=9))
    assert "x must be" in _error(lin(x=None))
    assert "x must be" in _error(lin(ldx=32))
    assert "workspace" in _error(lin(ws=None))
    assert "workspace" in _error(lin(size=need - 1))
    assert "workspace" in _error(lin(ws=ctypes.c_void_p(272)))
    assert lin(m=0) == 0


def _layer(**kw):
    d = _lib.MoeLayerFp4Desc()
    d.struct_size = ctypes.sizeof(_lib.MoeLayerFp4Desc)
    for name in ("x", "logits", "w_gate_up", "gate_up_scales", "w_down", "down_scales", "out"):
        setattr(d, name, 256)
    d.tokens, d.num_experts, d.top_k, d.hidden, d.ffn = 2, 4, 2, 64, 128
    for name, v in kw.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("change, words", [
    (dict(struct_size=8), "struct_size"), (dict(format=2), "format"), (dict(tokens=33), "tokens=33"), (dict(tokens=-1), "tokens=-1"),
    (dict(num_experts=257), "num_experts=257"), (dict(num_experts=0), "num_experts=0"), (dict(top_k=5), "top_k=5"),
    (dict(top_k=9, num_experts=16), "top_k=9"), (dict(top_k=0), "top_k=0"), (dict(hidden=96), "multiples of 64"),
    (dict(ffn=32), "multiples of 64"), (dict(hidden=0), "multiples of 64"), (dict(gate_up_tensor_scale=256), "tensor scale"),
    (dict(down_tensor_scale=256), "tensor scale"), (dict(x=None), "NULL"), (dict(logits=None), "NULL"), (dict(w_down=264), "aligned"),
    (dict(out=264), "aligned"), (dict(logits=258), "aligned"),
])
def test_moe_refusals(change, words):
    lib = _lib.load()
    ws = ctypes.c_void_p(1024)
    assert words in _error(lib.rb200_moe_layer_fp4(ctypes.byref(_layer(**change)), ws, 1 << 20, None))


def test_moe_workspace_refusals():
    lib, ws = _lib.load(), ctypes.c_void_p(1024)
    need = lib.rb200_moe_layer_fp4_workspace_bytes(2, 2, 64, 128)
    assert "NULL" in _error(lib.rb200_moe_layer_fp4(ctypes.byref(_layer()), None, need, None))
    assert "workspace" in _error(lib.rb200_moe_layer_fp4(ctypes.byref(_layer()), ws, need - 1, None))
    assert "aligned" in _error(lib.rb200_moe_layer_fp4(ctypes.byref(_layer()), ctypes.c_void_p(1032), need, None))
    assert lib.rb200_moe_layer_fp4(ctypes.byref(_layer(tokens=0)), ws, need, None) == 0


def test_python_refusals():
    x = torch.zeros(4, 64).half()
    with pytest.raises(ValueError, match="mx"):
        ops.encode_fp4(x, "fp4")
    with pytest.raises(ValueError, match="k % 32"):
        ops.encode_fp4(torch.zeros(4, 48).half(), "mx")
    with pytest.raises(ValueError, match="batch"):
        ops.encode_fp4(torch.zeros(64).half(), "mx")
    with pytest.raises(relax_b200.RB200Error, match="CUDA device"):
        ops.encode_fp4(x, "mx")
    with pytest.raises(relax_b200.RB200Error, match="float16"):
        ops.encode_fp4(torch.zeros(4, 64, dtype=torch.int32), "mx")
    with pytest.raises(TypeError, match="dtype"):
        ops.decode_fp4(x, x, "mx", dtype="half")
    c = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="codes"):
        ops.gemm_fp4(c[0], c, c, c, "mx")
    with pytest.raises(relax_b200.RB200Error, match="CUDA device"):
        ops.linear_fp4(x, c, torch.zeros(1, 1, 512, dtype=torch.uint8), "mx")


def test_an_empty_batch_has_a_residual_without_an_address():
    lib = _lib.load()
    assert lib.rb200_gemm_fp4(ctypes.byref(_desc(m=0, binary_op=1)), None) == 0
    assert lib.rb200_gemm_fp4(ctypes.byref(_desc(m=0, binary_op=3)), None) == -1
