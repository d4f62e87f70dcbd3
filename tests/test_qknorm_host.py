"""qk_norm_rope's refusals: the wrapper's checks and the C ABI's, before anything reaches a GPU."""

import ctypes

import pytest
import torch

from solarwm_amd import _lib, qk_norm_rope

D = 128


def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def _tables(rows, cols):
    return torch.zeros(rows, cols), torch.zeros(rows, cols)


@pytest.mark.parametrize("text,kw", [
    (r"q must be \[B, L, H, 128\]", dict(q=_x(1, 4, 2, 64))),
    (r"q must be \[B, L, H, 128\]", dict(q=_x(4, 2, D))),
    ("q dtype", dict(q=_x(1, 4, 2, D, dtype=torch.float64))),
    ("share dtype", dict(k=_x(1, 4, 2, D, dtype=torch.float16))),
    ("share dtype", dict(k=_x(1, 5, 2, D))),
    ("no heads", dict(q=_x(1, 4, 0, D))),
    ("no heads", dict(k=_x(1, 4, 0, D))),
    ("cos and sin together", dict(sin=None)),
    ("columns", dict(cos=_tables(4, 12)[0], sin=_tables(4, 12)[1])),
    ("columns", dict(cos=_tables(4, 72)[0], sin=_tables(4, 72)[1])),
    (r"must be \[positions, pairs\]", dict(cos=_tables(4, 16)[0])),
    ("float32", dict(cos=_tables(4, 64)[0].half(), sin=_tables(4, 64)[1].half())),
    ("share strides", dict(cos=torch.zeros(64, 4).t(), sin=torch.zeros(64, 4).t())),
    ("no gradient", dict(cos=_tables(4, 64)[0].requires_grad_())),
    ("do not lie", dict(position0=1)),
    ("do not lie", dict(position0=-1)),
    ("positions must be int32", dict(positions=torch.zeros(4))),
    (r"positions must be \[4\]", dict(positions=torch.zeros(3, dtype=torch.int32))),
    ("positions without", dict(cos=None, sin=None, positions=torch.zeros(4, dtype=torch.int32))),
    (r"norm_q weight must be \[128\]", dict(norm_q=(torch.zeros(2 * D), 1e-6))),
    ("norm_k weight", dict(norm_k=(torch.zeros(D, dtype=torch.float64), 1e-6))),
    ("contiguous", dict(norm_q=(torch.zeros(2 * D)[::2], 1e-6))),
    ("norm_k without k", dict(k=None, norm_k=(None, 1e-6))),
    ("GPU tensor", dict()),
])
def test_refusals(text, kw):
    args = dict(q=_x(1, 4, 2, D), k=_x(1, 4, 2, D), cos=_tables(4, 64)[0], sin=_tables(4, 64)[1])
    args.update(kw)
    q, k, cos, sin = (args.pop(n) for n in ("q", "k", "cos", "sin"))
    with pytest.raises(ValueError, match=text):
        qk_norm_rope(q, k, cos, sin, **args)


def _desc(**kw):
    p = 0x1000
    d = _lib.QkNormRopeDesc(dtype=_lib.SKV_BF16, batch=1, rows=4, head_dim=D, cos=p, sin=p, table_stride=64,
                            table_rows=4, half=64)
    for s in (d.q, d.k):
        s.x, s.out, s.grad, s.heads, s.norm = p, 0x100000, p, 2, 1
        s.x_st = s.out_st = s.grad_st = 2 * D
        s.x_sh = s.out_sh = s.grad_sh = D
    for name, value in kw.items():
        side, _, field = name.rpartition("_side_")
        setattr(getattr(d, side) if side else d, field if side else name, value)
    return d


@pytest.mark.parametrize("entry", ["skv_qk_norm_rope", "skv_qk_norm_rope_grad"])
@pytest.mark.parametrize("status,text,kw", [
    (_lib.SKV_E_UNSUPPORTED, b"head_dim", dict(head_dim=64)),
    (_lib.SKV_E_UNSUPPORTED, b"dtype", dict(dtype=_lib.SKV_FP8_E4M3)),
    (_lib.SKV_E_ARG, b"bad sizes", dict(rows=-1)),
    (_lib.SKV_E_ARG, b"rotation", dict(half=12)),
    (_lib.SKV_E_ARG, b"rotation", dict(half=0)),
    (_lib.SKV_E_ARG, b"rotation", dict(sin=None)),
    (_lib.SKV_E_ARG, b"row stride", dict(table_stride=63)),
    (_lib.SKV_E_ARG, b"row stride", dict(table_rows=0)),
    (_lib.SKV_E_ARG, b"row stride", dict(cos=0x1004)),
    (_lib.SKV_E_ARG, b"q tensors must be 16-byte", dict(q_side_x=0x1002)),
    (_lib.SKV_E_ARG, b"q tensors must be 16-byte", dict(q_side_x_st=-8)),
    (_lib.SKV_E_ARG, b"k tensors must be 16-byte", dict(k_side_out_sh=4)),
    (_lib.SKV_E_ARG, b"k has -1 heads", dict(k_side_heads=-1)),
    (_lib.SKV_E_ARG, b"q has 0 heads", dict(q_side_heads=0)),
    (_lib.SKV_E_ARG, b"norm weight", dict(q_side_weight=0x1002)),
    (_lib.SKV_E_ARG, b"eps", dict(q_side_eps=-1.0)),
    (_lib.SKV_E_ARG, b"overlaps", dict(q_side_out=0x1100)),
    (_lib.SKV_E_ARG, b"too many rows", dict(batch=4, rows=1 << 30, q_side_x_st=0, q_side_out_st=0,
                                             k_side_x_st=0, k_side_out_st=0)),
])
def test_descriptor_errors_do_not_launch(entry, status, text, kw):
    lib = _lib.load()
    assert getattr(lib, entry)(ctypes.byref(_desc(**kw)), None) == status
    assert text in lib.skv_last_error()


def test_gradient_errors_do_not_launch():
    lib = _lib.load()
    size = ctypes.c_int64(0)
    d = _desc(q_side_grad=None)
    assert lib.skv_qk_norm_rope_grad(ctypes.byref(d), None) == _lib.SKV_E_ARG
    assert b"q tensors" in lib.skv_last_error()
    d = _desc(q_side_grad_weight=0x1000)
    assert lib.skv_qk_norm_rope_grad_workspace(ctypes.byref(d), ctypes.byref(size)) == 0
    assert size.value == D * 4  # 4 tokens of one head block: one workgroup's partial sums
    assert lib.skv_qk_norm_rope_grad(ctypes.byref(d), None) == _lib.SKV_E_ARG
    assert b"workspace" in lib.skv_last_error()
    d = _desc(q_side_grad_weight=0x1000, q_side_norm=0)
    assert lib.skv_qk_norm_rope_grad(ctypes.byref(d), None) == _lib.SKV_E_ARG
    assert b"grad_weight" in lib.skv_last_error()
    assert lib.skv_qk_norm_rope(None, None) == _lib.SKV_E_ARG


@pytest.mark.parametrize("entry", ["skv_qk_norm_rope", "skv_qk_norm_rope_grad"])
@pytest.mark.parametrize("kw", [dict(batch=(1 << 31) - 1, rows=(1 << 31) - 1), dict(batch=1, rows=1 << 28),
                                dict(batch=1, rows=1 << 30, q_side_heads=(1 << 31) - 1, q_side_x_sh=0,
                                     q_side_out_sh=0)])
def test_sizes_past_a_launch(entry, kw):
    lib = _lib.load()
    d = _desc(q_side_x_st=0, q_side_out_st=0, k_side_x_st=0, k_side_out_st=0, **kw)
    assert getattr(lib, entry)(ctypes.byref(d), None) == _lib.SKV_E_ARG
    assert b"too many rows" in lib.skv_last_error()
