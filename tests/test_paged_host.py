"""Refusals of append_pages, attend_shared and history_pages: the wrappers' checks and the C ABI's,
before anything reaches a GPU."""

import ctypes

import pytest
import torch

from solarwm_amd import (RopeConfig, _lib, append_pages, attend_shared, history_pages,
                         make_kv_cache_allocator)

D = 128
BF = torch.bfloat16


def _x(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _args(**kw):
    a = dict(k=_x(2, 3, 2, D), v=_x(2, 3, 2, D), q=_x(2, 3, 4, D), kpool=_x(5, 1, 2, 64, D),
             vpool=_x(5, 1, 2, D, 64), tables=torch.zeros(2, 2, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32), page_tokens=50)
    a.update(kw)
    return a


COMMON = [
    ("pools must be K", dict(kpool=_x(5, 2, 2, 64, D))),
    ("do not match page_tokens=65", dict(page_tokens=65)),
    ("do not match", dict(vpool=_x(5, 1, 2, 64, D))),
    ("page_tokens must be positive", dict(page_tokens=0)),
    ("pools are", dict(vpool=_x(5, 1, 2, D, 64, dtype=torch.float16))),
    ("pools must be contiguous", dict(kpool=_x(5, 1, 2, D, 64).transpose(3, 4))),
    ("no pages", dict(kpool=_x(0, 1, 2, 64, D), vpool=_x(0, 1, 2, D, 64))),
    ("tables must be int32", dict(tables=torch.zeros(2, 2, dtype=torch.int64))),
    ("tables must be int32", dict(tables=torch.zeros(3, 2, dtype=torch.int32))),
    ("contiguous in their last", dict(tables=torch.zeros(2, 4, dtype=torch.int32)[:, ::2])),
    ("lengths must be int32", dict(lengths=torch.zeros(2))),
    ("lengths must be int32", dict(lengths=torch.zeros(3, dtype=torch.int32))),
    ("lengths must be contiguous", dict(lengths=torch.zeros(4, dtype=torch.int32)[::2])),
    ("new_lens must be int32", dict(new_lens=torch.zeros(2, dtype=torch.int64))),
    ("GPU tensor", dict()),
]


@pytest.mark.parametrize("text,kw", COMMON + [
    (r"k must be \[B, L, H, 128\]", dict(k=_x(2, 3, 2, 64))),
    ("k dtype", dict(k=_x(2, 3, 2, D, dtype=torch.float32))),
    ("k and v must share", dict(v=_x(2, 3, 1, D))),
    ("k / v have 2 heads", dict(kpool=_x(5, 1, 3, 64, D), vpool=_x(5, 1, 3, D, 64))),
    ("q must share", dict(q=_x(2, 4, 4, D))),
    ("q must share", dict(q=_x(2, 3, 0, D))),
    ("cos and sin together", dict(cos=torch.zeros(4, 64))),
    ("positions without", dict(positions=torch.zeros(3, dtype=torch.int32))),
    ("positions must be", dict(cos=torch.zeros(4, 64), sin=torch.zeros(4, 64), positions=torch.zeros(3))),
    ("norm_k weight", dict(norm_k=(torch.zeros(2 * D), 1e-6))),
    ("norm_q / out without q", dict(q=None, norm_q=(None, 1e-6))),
    ("out must match", dict(out=_x(2, 3, 2, D))),
    ("must not be expanded", dict(out=_x(1, 3, 4, D).expand(2, 3, 4, D))),
    ("contiguous in its last", dict(v=_x(2, 3, D, 2).transpose(2, 3))),
])
def test_append_refusals(text, kw):
    a = _args(**kw)
    with pytest.raises(ValueError, match=text):
        append_pages(a.pop("k"), a.pop("v"), a.pop("kpool"), a.pop("vpool"), a.pop("tables"), a.pop("lengths"), **a)


@pytest.mark.parametrize("text,kw", COMMON + [
    (r"q must be \[B, L, H, 128\]", dict(q=_x(2, 4, D))),
    ("q dtype", dict(q=_x(2, 3, 4, D, dtype=torch.float32))),
    ("no multiple", dict(q=_x(2, 3, 3, D))),
    ("softmax_scale", dict(softmax_scale=0.0)),
    ("softmax_scale", dict(softmax_scale=float("nan"))),
    ("without prefix_pages", dict(prefix_tokens=10)),
    ("do not lie in 1 pages", dict(prefix_tokens=51, prefix_pages=torch.zeros(1, dtype=torch.int32))),
    ("do not lie", dict(prefix_tokens=-1, prefix_pages=torch.zeros(1, dtype=torch.int32))),
    ("prefix_pages must be int32", dict(prefix_tokens=1, prefix_pages=torch.zeros(1))),
    ("prefix pools have 1 heads", dict(prefix_tokens=1, prefix_pages=torch.zeros(1, dtype=torch.int32),
                                       prefix_pools=(_x(1, 1, 1, 64, D), _x(1, 1, 1, D, 64), 64))),
    ("prefix pool shapes", dict(prefix_tokens=1, prefix_pages=torch.zeros(1, dtype=torch.int32),
                                prefix_pools=(_x(1, 1, 2, 64, D), _x(1, 1, 2, D, 64), 65))),
    ("out must match", dict(out=_x(2, 3, 4, D, dtype=torch.float16))),
    ("must not be expanded", dict(out=_x(2, 3, 1, D).expand(2, 3, 4, D))),
])
def test_attend_refusals(text, kw):
    a = _args(**kw)
    a.pop("k"), a.pop("v")
    with pytest.raises(ValueError, match=text):
        attend_shared(a.pop("q"), a.pop("kpool"), a.pop("vpool"), a.pop("tables"), a.pop("lengths"), **a)


def _cache(batch=1, dtype=BF, **kw):
    return make_kv_cache_allocator(num_layers=1, num_heads=1, head_dim=D, frame_sequence_length=64,
                                   local_attn_size=2, **kw)(batch, dtype=dtype, device="cpu")[0]


def test_history_refusals():
    pages, tokens, pools = history_pages(_cache())
    assert pages.tolist() == [] and tokens == 0 and pools[2] == 64
    with pytest.raises(ValueError, match="batch of one"):
        history_pages(_cache(batch=2))
    with pytest.raises(ValueError, match="rotates them on load"):
        history_pages(_cache(rope=RopeConfig(grid_hw=(8, 8))))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        history_pages(_cache(dtype=torch.float32))


def _desc(kind, **kw):
    p = 0x1000
    d = kind(dtype=_lib.SKV_BF16, n_pages=4, page_tokens=64, batch=2, rows=3, q_heads=4, kv_heads=2,
             head_dim=D, k_pool=p, v_pool=p, tables=p, table_stride=2, table_width=2, lengths=p, q=p)
    if kind is _lib.AppendPagesDesc:
        d.k = d.v = d.q_out = p
    else:
        d.out, d.softmax_scale = p, 0.1
    for name, value in kw.items():
        setattr(d, name, value)
    return d


SIZES = [
    (_lib.SKV_E_UNSUPPORTED, b"head_dim", dict(head_dim=64)),
    (_lib.SKV_E_UNSUPPORTED, b"dtype", dict(dtype=_lib.SKV_F32)),
    (_lib.SKV_E_ARG, b"bad sizes", dict(batch=-1)),
    (_lib.SKV_E_ARG, b"bad sizes", dict(kv_heads=0)),
    (_lib.SKV_E_ARG, b"bad pool", dict(n_pages=0)),
    (_lib.SKV_E_ARG, b"bad pool", dict(page_tokens=-1)),
    (_lib.SKV_E_ARG, b"page tables", dict(tables=None)),
    (_lib.SKV_E_ARG, b"page tables", dict(lengths=None)),
    (_lib.SKV_E_ARG, b"page tables", dict(table_width=1 << 30)),
    (_lib.SKV_E_ARG, b"pools must be", dict(k_pool=0x1008)),
    (_lib.SKV_E_ARG, b"16-byte aligned", dict(q=0x1004)),
    (_lib.SKV_E_ARG, b"multiples of", dict(q_st=12)),
]


@pytest.mark.parametrize("status,text,kw", SIZES + [
    (_lib.SKV_E_ARG, b"multiples of", dict(v_sh=4)),
    (_lib.SKV_E_ARG, b"rotation", dict(half=8)),
    (_lib.SKV_E_ARG, b"row stride", dict(half=8, cos=0x1000, sin=0x1000, cos_stride=8)),
    (_lib.SKV_E_ARG, b"too many rows", dict(rows=1 << 29)),
    (_lib.SKV_E_ARG, b"norms need", dict(norm_k=_lib.HeadNorm(norm=1, eps=-1.0))),
    (_lib.SKV_E_ARG, b"norms need", dict(norm_q=_lib.HeadNorm(norm=1, weight=0x1004))),
])
def test_append_descriptor_errors_do_not_launch(status, text, kw):
    lib = _lib.load()
    assert lib.skv_append_pages(ctypes.byref(_desc(_lib.AppendPagesDesc, **kw)), None) == status
    assert text in lib.skv_last_error()
    assert lib.skv_append_pages(None, None) == _lib.SKV_E_ARG


@pytest.mark.parametrize("status,text,kw", SIZES + [
    (_lib.SKV_E_ARG, b"bad sizes", dict(q_heads=3)),
    (_lib.SKV_E_ARG, b"multiples of", dict(out_sb=4)),
    (_lib.SKV_E_ARG, b"bad prefix", dict(prefix_tokens=5)),
    (_lib.SKV_E_ARG, b"bad prefix", dict(prefix_tokens=-5)),
    (_lib.SKV_E_ARG, b"softmax_scale", dict(softmax_scale=0.0)),
    (_lib.SKV_E_ARG, b"too many query rows", dict(rows=1 << 29)),
    (_lib.SKV_E_ARG, b"workspace", dict(prefix_tokens=64, prefix_k_pool=0x1000, prefix_v_pool=0x1000,
                                        prefix_n_pages=1, prefix_page_tokens=64, prefix_pages=0x1000)),
])
def test_attend_descriptor_errors_do_not_launch(status, text, kw):
    lib = _lib.load()
    d = _desc(_lib.AttendSharedDesc, **kw)
    assert lib.skv_attend_shared(ctypes.byref(d), None) == status
    assert text in lib.skv_last_error()
    assert lib.skv_attend_shared(None, None) == _lib.SKV_E_ARG


PREFIX = dict(prefix_tokens=64, prefix_k_pool=0x1000, prefix_v_pool=0x1000, prefix_n_pages=1,
              prefix_page_tokens=64, prefix_pages=0x1000)


@pytest.mark.parametrize("kw", [dict(batch=0), dict(rows=0), dict(batch=1, rows=0), dict(batch=0, **PREFIX),
                                dict(rows=0, **PREFIX), dict(batch=1, rows=0, **PREFIX)])
def test_nothing_to_do(kw):
    """No sequences or no rows: nothing is launched, with and without a prefix."""
    lib, size = _lib.load(), ctypes.c_int64(-1)
    d = _desc(_lib.AttendSharedDesc, **kw)
    assert lib.skv_attend_shared_workspace(ctypes.byref(d), ctypes.byref(size)) == 0 and size.value == 0
    assert lib.skv_attend_shared(ctypes.byref(d), None) == 0
    d = _desc(_lib.AppendPagesDesc, **{k: v for k, v in kw.items() if not k.startswith("prefix")})
    assert lib.skv_append_pages(ctypes.byref(d), None) == 0


MOST = (1 << 31) - 1


@pytest.mark.parametrize("kw", [
    dict(batch=MOST, rows=MOST), dict(batch=MOST, rows=MOST, q_heads=MOST, kv_heads=MOST),
    dict(batch=1, rows=MOST, q_heads=MOST, kv_heads=MOST), dict(batch=1 << 28, rows=1, q_heads=2, kv_heads=1),
    dict(batch=MOST, rows=1, q_heads=MOST, kv_heads=1, page_tokens=1),
])
def test_sizes_past_a_launch(kw):
    """Sizes that no launch takes are refused, whatever their products wrap to."""
    lib = _lib.load()
    for kind, entry in ((_lib.AttendSharedDesc, "skv_attend_shared"), (_lib.AppendPagesDesc, "skv_append_pages")):
        d = _desc(kind, **kw)
        assert getattr(lib, entry)(ctypes.byref(d), None) == _lib.SKV_E_ARG
        assert b"too many" in lib.skv_last_error()
