"""RMS norm of every query and key head with the position rotation in the same pass, and its
gradient.

The H3 blocks normalise each 128-channel head of q and k and rotate it before attention
(minimax_h3/fused_ops.py:1-16, forward and backward).  Here both heads' tensors go through one
launch, which reads them once and writes them once; the values are normalised, weighted and
rotated in fp32 and rounded once, on the way out.  (The Wan blocks normalise a token's whole
``H * D`` row instead: ``kernels.rms_rows`` and ``norm_q=`` / ``norm_k=`` of ``attend_cached``.)
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, kernels

HEAD_DIM = kernels.HEAD_DIM
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def launch(entry: str, desc, device: torch.device) -> None:
    """Call a descriptor entry point on ``device``'s current stream, with ``device`` current."""
    fn = getattr(_lib.load(), entry)
    index = kernels._device_index(device)
    if torch._C._cuda_getDevice() == index:
        status = fn(ctypes.byref(desc), torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(ctypes.byref(desc), torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(entry, status)


def head_norm_spec(name: str, norm) -> tuple[torch.Tensor | None, float]:
    """(weight [128] or None, eps) of a norm given as an object with ``weight`` and ``eps`` or as
    a ``(weight, eps)`` pair."""
    weight, eps = norm if isinstance(norm, tuple) else (norm.weight, norm.eps)
    if weight is not None:
        if weight.shape != (HEAD_DIM,) or weight.dtype not in _FLOATS:
            raise ValueError(f"{name} weight must be [{HEAD_DIM}] (one head), float32, bfloat16 or "
                             f"float16; got {weight.dtype} {tuple(weight.shape)}")
        if not weight.is_contiguous():
            raise ValueError(f"{name} weight must be contiguous")
    return weight, float(eps)


def strides(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    """(sb, st, sh) of a [B, L, H, 128] tensor with unit channel stride; 0 where there is one step."""
    sb, st, sh, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    b, l, h, _ = t.shape
    return sb if b > 1 else 0, st if l > 1 else 0, sh if h > 1 else 0


def check_heads(name: str, t: torch.Tensor, dtypes) -> None:
    shape = t.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM:
        raise ValueError(f"{name} must be [B, L, H, {HEAD_DIM}], got {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype {t.dtype} unsupported ({', '.join(map(str, dtypes))})")


def check_tables(cos, sin) -> None:
    if (cos is None) != (sin is None):
        raise ValueError("give cos and sin together")
    if cos is None:
        return
    shape, stride = cos.shape, cos.stride()
    if len(shape) != 2 or sin.shape != shape:
        raise ValueError(f"cos / sin must be [positions, pairs], got {tuple(cos.shape)} / {tuple(sin.shape)}")
    if shape[1] % 8 or not 8 <= shape[1] <= HEAD_DIM // 2:
        raise ValueError(f"cos / sin need 8, 16 .. {HEAD_DIM // 2} columns (one per rotated pair), got {shape[1]}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos / sin must be float32")
    if stride[1] != 1 or sin.stride() != stride:
        raise ValueError("cos and sin must share strides, with unit column stride")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise ValueError("cos / sin take no gradient")


def check_positions(positions, batch: int, rows: int) -> tuple[int, int]:
    """(batch stride, token stride) of integer positions [L] or [B, L]."""
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if tuple(positions.shape) == (rows,):
        return 0, positions.stride(0)
    if tuple(positions.shape) == (batch, rows):
        return positions.stride(0), positions.stride(1)
    raise ValueError(f"positions must be [{rows}] or [{batch}, {rows}], got {tuple(positions.shape)}")


def same_device(names: tuple[str, ...], tensors: tuple) -> None:
    """Every tensor that is given is on the GPU of the first."""
    index = tensors[0].get_device()  # -1: not on a GPU
    if index >= 0:
        for t in tensors:
            if t is not None and t.get_device() != index:
                break
        else:
            return
    device = tensors[0].device
    for name, t in zip(names, tensors):
        if t is not None:
            kernels._require_cuda(name, t)
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, expected {device}")


def empty_as(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _desc(q, k, wq, wk, cos, sin, positions, meta) -> _lib.QkNormRopeDesc:
    """Descriptor of the inputs; the caller adds out (and grad, grad_weight, workspace)."""
    norm_q, eps_q, norm_k, eps_k, position0, interleaved = meta
    b, l, h, _ = q.shape
    d = _lib.QkNormRopeDesc(dtype=kernels.dtype_code(q.dtype), batch=b, rows=l, head_dim=HEAD_DIM,
                            interleaved=interleaved, position0=position0)
    for s, x, w, norm, eps in ((d.q, q, wq, norm_q, eps_q), (d.k, k, wk, norm_k, eps_k)):
        if x is None:
            continue
        s.x = x.data_ptr()
        s.x_sb, s.x_st, s.x_sh = strides("q / k", x)
        s.heads, s.norm, s.eps = x.shape[2], norm, eps
        if w is not None:
            s.weight, s.weight_dtype = w.data_ptr(), kernels.dtype_code(w.dtype)
    if cos is not None:
        d.cos, d.sin, d.half = cos.data_ptr(), sin.data_ptr(), cos.shape[1]
        d.table_rows = cos.shape[0]
        d.table_stride = cos.stride(0) if cos.shape[0] > 1 else cos.shape[1]
    if positions is not None:
        d.positions, d.pos_is_int64 = positions.data_ptr(), positions.dtype == torch.int64
        d.pos_sb, d.pos_st = check_positions(positions, b, l)
    return d


def _set_out(side, x: torch.Tensor) -> None:
    side.out = x.data_ptr()
    b, l, h, _ = x.shape
    side.out_sb, side.out_st, side.out_sh = l * h * HEAD_DIM, h * HEAD_DIM, HEAD_DIM


def _forward(q, k, wq, wk, cos, sin, positions, meta):
    zq, zk = empty_as(q), None if k is None else empty_as(k)
    if q.numel() == 0:
        return zq, zk
    d = _desc(q, k, wq, wk, cos, sin, positions, meta)
    _set_out(d.q, zq)
    if k is not None:
        _set_out(d.k, zk)
    launch("skv_qk_norm_rope", d, q.device)
    return zq, zk


def _readable(g: torch.Tensor) -> torch.Tensor:
    """``g`` itself where the kernel can read it in place, else a contiguous copy."""
    if g.stride(3) == 1 and g.data_ptr() % 16 == 0 and all(
            s % 8 == 0 for s, n in zip(g.stride()[:3], g.shape[:3]) if n > 1):
        return g
    return g.clone(memory_format=torch.contiguous_format)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, meta):
        zq, zk = _forward(q, k, wq, wk, cos, sin, positions, meta)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        ctx.meta = meta
        return zq, zk

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        dq, dk = empty_as(q), None if k is None else empty_as(k)
        need = ctx.needs_input_grad
        dwq = torch.empty_like(wq) if need[2] else None
        dwk = torch.empty_like(wk) if need[3] else None
        if q.numel() == 0:
            for t in (dwq, dwk):
                if t is not None:
                    t.zero_()
            return dq, dk, dwq, dwk, None, None, None, None
        d = _desc(q, k, wq, wk, cos, sin, positions, ctx.meta)
        keep = []
        for s, g, dx, w, dw in ((d.q, gq, dq, wq, dwq), (d.k, gk, dk, wk, dwk)):
            if dx is None:
                continue
            g = _readable(g)
            keep.append(g)
            s.grad = g.data_ptr()
            s.grad_sb, s.grad_st, s.grad_sh = strides("gradient", g)
            _set_out(s, dx)
            if dw is not None:
                s.grad_weight, s.grad_weight_dtype = dw.data_ptr(), kernels.dtype_code(dw.dtype)
        if dwq is not None or dwk is not None:
            size = ctypes.c_int64(0)
            status = _lib.load().skv_qk_norm_rope_grad_workspace(ctypes.byref(d), ctypes.byref(size))
            if status:
                _lib.check("skv_qk_norm_rope_grad_workspace", status)
            # a block of this call's own: two graphs captured on one stream may replay side by side
            ws = torch.empty(size.value, dtype=torch.uint8, device=q.device)
            d.workspace, d.workspace_bytes = ws.data_ptr(), size.value
            keep.append(ws)
        launch("skv_qk_norm_rope_grad", d, q.device)
        del keep
        return dq, dk, dwq, dwk, None, None, None, None


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor | None,
    cos: torch.Tensor | None,
    sin: torch.Tensor | None,
    *,
    norm_q=None,
    norm_k=None,
    positions: torch.Tensor | None = None,
    position0: int = 0,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Normalise every 128-channel head of ``q`` [B, L, Hq, 128] and ``k`` [B, L, Hk, 128] (or
    None) over its own channels and rotate it to its token's position; returns new tensors of the
    inputs' dtype (bfloat16, float16 or float32, the same for both).  Differentiable in q, k and
    the weights; the weights' gradients are summed in a fixed order.

    ``norm_q`` / ``norm_k``: a module with ``weight`` [128] (or None) and ``eps``, or a ``(weight,
    eps)`` pair; None leaves the tensor unnormalised.  ``cos`` / ``sin`` float32 [positions, r / 2]
    (8, 16 .. 64 columns; both None: no rotation) turn the first r channels of a head, neighbouring
    channels with ``interleaved`` and channels (i, i + r / 2) without.  A token's table row is
    ``position0`` plus ``positions`` (int32 or int64, [L] or [B, L]), by default its index in the
    sequence; channels turned by a row outside the table come back as NaN.

    q and k may be slices of one projection: any strides that are multiples of 8 elements with a
    unit channel stride and 16-byte alignment."""
    check_heads("q", q, _FLOATS)
    if k is not None:
        check_heads("k", k, _FLOATS)
        if k.dtype != q.dtype or k.shape[:2] != q.shape[:2]:
            raise ValueError(f"q and k must share dtype, batch and length, got {q.dtype} {tuple(q.shape)} / "
                             f"{k.dtype} {tuple(k.shape)}")
        if k.shape[2] == 0:
            raise ValueError("k has no heads")
    elif norm_k is not None:
        raise ValueError("norm_k without k")
    if q.shape[2] == 0:
        raise ValueError("q has no heads")
    check_tables(cos, sin)
    wq, eps_q = head_norm_spec("norm_q", norm_q) if norm_q is not None else (None, 0.0)
    wk, eps_k = head_norm_spec("norm_k", norm_k) if norm_k is not None else (None, 0.0)
    position0 = int(position0)
    if positions is not None:
        if cos is None:
            raise ValueError("positions without cos and sin")
        check_positions(positions, q.shape[0], q.shape[1])
    elif cos is not None and not 0 <= position0 <= cos.shape[0] - q.shape[1]:
        raise ValueError(f"positions {position0} .. {position0 + q.shape[1] - 1} do not lie in a table of "
                         f"{cos.shape[0]} rows")
    same_device(("q", "k", "cos", "sin", "norm_q", "norm_k", "positions"),
                (q, k, cos, sin, wq, wk, positions))
    meta = (norm_q is not None, eps_q, norm_k is not None, eps_k, position0, bool(interleaved))
    if torch.is_grad_enabled() and (
            q.requires_grad or (k is not None and k.requires_grad)
            or (wq is not None and wq.requires_grad) or (wk is not None and wk.requires_grad)):
        return _QkNormRope.apply(q, k, wq, wk, cos, sin, positions, meta)
    return _forward(q, k, wq, wk, cos, sin, positions, meta)
