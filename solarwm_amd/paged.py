"""Sequences that share a history: paged caches and attention over one prefix for a whole batch.

Several rollouts that continue one history (other actions, other prompts, other seeds) see the
same keys up to the point where they part.  Here that history is kept once, in pages, and each
sequence goes on in pages of its own:

* a page is a frame slot with a batch of one, ``kernels.new_pools(n_pages, 1, heads, page_tokens,
  dtype, device)``: K ``[n_pages, 1, H, Tp, 128]``, V ``[n_pages, 1, H, 128, Tp]`` transposed, with
  ``page_tokens`` tokens in use (attention works on 64 keys of a page at a time: multiples of 64 cost
  least); the other functions on pools (``kernels.gather_frames``, ...) take
  them as they are, and a frame-slot cache with a batch of one is such a pool itself
  (:func:`history_pages`);
* ``tables`` (int32 ``[B, W]`` on the GPU) names each sequence's pages in order, ``lengths`` (int32
  ``[B]`` on the GPU) its own tokens including those of the current call, and ``new_lens`` (int32
  ``[B]``, optional) how many of a padded call's rows are new tokens of it (the first ones);
* an entry outside the pool's pages is a page that is not there: nothing is written to it and its
  keys are not seen.

A step of such a batch is :func:`append_pages` (keys normalised and rotated on the way, the queries
with them), then :func:`attend_shared`.  Nothing is read back to the host, so a step can be captured
into a HIP graph and replayed while ``lengths`` and ``tables`` change on the GPU.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, kernels
from .cache import SlotKVCache
from .qknorm import (HEAD_DIM, check_heads, check_positions, check_tables, empty_as, head_norm_spec,
                     launch, same_device, strides)

_HALVES = (torch.bfloat16, torch.float16)


def _check_pools(what: str, kpool: torch.Tensor, vpool: torch.Tensor, page_tokens: int,
                 dtype: torch.dtype) -> tuple[int, int]:
    """(pages, heads) of a pool pair with a batch of one."""
    if page_tokens <= 0:
        raise ValueError(f"{what}page_tokens must be positive, got {page_tokens}")
    tp = kernels.padded_tokens(page_tokens)
    shape = kpool.shape
    if len(shape) != 5 or shape[1] != 1:
        raise ValueError(f"{what}pools must be K [pages, 1, H, Tp, 128] / V [pages, 1, H, 128, Tp], got "
                         f"{tuple(shape)}")
    n, _, h, rows, width = shape
    if rows != tp or width != HEAD_DIM or vpool.shape != (n, 1, h, HEAD_DIM, tp):
        raise ValueError(f"{what}pool shapes {tuple(kpool.shape)} / {tuple(vpool.shape)} do not match "
                         f"page_tokens={page_tokens} (Tp = {tp})")
    if kpool.dtype != dtype or vpool.dtype != dtype:
        raise ValueError(f"{what}pools are {kpool.dtype} / {vpool.dtype}, the tokens {dtype}")
    if not (kpool.is_contiguous() and vpool.is_contiguous()):
        raise ValueError(f"{what}pools must be contiguous")
    if n == 0:
        raise ValueError(f"{what}pools have no pages")
    return n, h


def _int32_vector(name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != (n,):
        raise ValueError(f"{name} must be int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _check_out(out: torch.Tensor, q: torch.Tensor) -> None:
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must match q's shape and dtype")
    if any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
        raise ValueError("out must not be expanded: its rows would lie on one another")


def _set_pages(d, kpool, vpool, n_pages, page_tokens, tables, lengths, new_lens, batch) -> None:
    """The fields that both descriptors share."""
    shape, stride = tables.shape, tables.stride()
    if tables.dtype != torch.int32 or len(shape) != 2 or shape[0] != batch:
        raise ValueError(f"tables must be int32 [{batch}, pages], got {tables.dtype} {tuple(shape)}")
    if shape[1] > 1 and stride[1] != 1:
        raise ValueError("tables must be contiguous in their last dimension")
    _int32_vector("lengths", lengths, batch)
    if new_lens is not None:
        _int32_vector("new_lens", new_lens, batch)
        d.new_lens = new_lens.data_ptr()
    d.k_pool, d.v_pool = kpool.data_ptr(), vpool.data_ptr()
    d.dtype, d.n_pages, d.page_tokens = kernels.dtype_code(kpool.dtype), n_pages, page_tokens
    d.tables, d.table_width = tables.data_ptr(), shape[1]
    d.table_stride = stride[0] if batch > 1 else 0
    d.lengths, d.head_dim = lengths.data_ptr(), HEAD_DIM


def append_pages(
    k: torch.Tensor,
    v: torch.Tensor,
    kpool: torch.Tensor,
    vpool: torch.Tensor,
    tables: torch.Tensor,
    lengths: torch.Tensor,
    *,
    page_tokens: int,
    new_lens: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    position0: int = 0,
    interleaved: bool = False,
    norm_q=None,
    norm_k=None,
    out: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write the new tokens ``k`` / ``v`` [B, L, H, 128] (bfloat16 or float16, the pools' dtype) to
    their pages, in one launch: row t of sequence b is its token ``lengths[b] - new_lens[b] + t``
    (``new_lens`` None: all L rows are new).  K is normalised over each head (``norm_k``) and rotated
    (``cos`` / ``sin``, ``interleaved``) as :func:`qk_norm_rope` does, rounded once; a token's table
    row is ``position0`` plus its own index, or plus ``positions`` (int32 or int64, [L] or [B, L])
    where given, so ``position0`` is the length of a shared prefix.

    ``q`` [B, L, Hq, 128] goes through ``norm_q`` and the same rotation; the result (or ``out``, which
    may be ``q`` itself and must not otherwise share memory with an input) is returned, with zeros in
    rows that are no new tokens.  No gradient is recorded.  Rows that are no new
    tokens and tokens whose page is not there leave the pools as they were.  Each page takes tokens of
    one sequence only; where two tokens of a call share a place, either's values may stay."""
    check_heads("k", k, _HALVES)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must share shape and dtype, got {k.dtype} {tuple(k.shape)} / {v.dtype} "
                         f"{tuple(v.shape)}")
    b, l, h, _ = k.shape
    n_pages, heads = _check_pools("", kpool, vpool, page_tokens, k.dtype)
    if h != heads:
        raise ValueError(f"k / v have {h} heads, the pools {heads}")
    check_tables(cos, sin)
    d = _lib.AppendPagesDesc(batch=b, rows=l, kv_heads=h, interleaved=bool(interleaved),
                             position0=int(position0))
    _set_pages(d, kpool, vpool, n_pages, page_tokens, tables, lengths, new_lens, b)
    wq = wk = None
    if norm_k is not None:
        wk, d.norm_k.eps = head_norm_spec("norm_k", norm_k)
        d.norm_k.norm = 1
        if wk is not None:
            d.norm_k.weight, d.norm_k.weight_dtype = wk.data_ptr(), kernels.dtype_code(wk.dtype)
    if q is not None:
        check_heads("q", q, _HALVES)
        if q.dtype != k.dtype or q.shape[:2] != k.shape[:2] or q.shape[2] == 0:
            raise ValueError(f"q must share k's dtype, batch and length, got {q.dtype} {tuple(q.shape)}")
        if out is None:
            out = empty_as(q)
        else:
            _check_out(out, q)
        d.q, d.q_out, d.q_heads = q.data_ptr(), out.data_ptr(), q.shape[2]
        d.q_sb, d.q_st, d.q_sh = strides("q", q)
        d.out_sb, d.out_st, d.out_sh = strides("out", out)
        if norm_q is not None:
            wq, d.norm_q.eps = head_norm_spec("norm_q", norm_q)
            d.norm_q.norm = 1
            if wq is not None:
                d.norm_q.weight, d.norm_q.weight_dtype = wq.data_ptr(), kernels.dtype_code(wq.dtype)
    elif norm_q is not None or out is not None:
        raise ValueError("norm_q / out without q")
    d.k, d.v = k.data_ptr(), v.data_ptr()
    d.k_sb, d.k_st, d.k_sh = strides("k", k)
    d.v_sb, d.v_st, d.v_sh = strides("v", v)
    if cos is not None:
        d.cos, d.sin = cos.data_ptr(), sin.data_ptr()
        d.table_rows, d.half = cos.shape
        d.cos_stride = cos.stride(0) if d.table_rows > 1 else d.half
    if positions is not None:
        if cos is None:
            raise ValueError("positions without cos and sin")
        d.pos_sb, d.pos_st = check_positions(positions, b, l)
        d.positions, d.pos_is_int64 = positions.data_ptr(), positions.dtype == torch.int64
    same_device(("k_pool", "v_pool", "k", "v", "q", "out", "tables", "lengths", "new_lens", "cos", "sin",
                 "positions", "norm_q", "norm_k"),
                (kpool, vpool, k, v, q, out, tables, lengths, new_lens, cos, sin, positions, wq, wk))
    if k.numel():
        launch("skv_append_pages", d, k.device)
    return out


def attend_shared(
    q: torch.Tensor,
    kpool: torch.Tensor,
    vpool: torch.Tensor,
    tables: torch.Tensor,
    lengths: torch.Tensor,
    *,
    page_tokens: int,
    prefix_pages: torch.Tensor | None = None,
    prefix_tokens: int = 0,
    prefix_pools: tuple[torch.Tensor, torch.Tensor, int] | None = None,
    new_lens: torch.Tensor | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(q kᵀ · scale) v for ``q`` [B, L, Hq, 128] (bfloat16 or float16) over the shared prefix
    and each sequence's own pages (already holding this call's tokens, see :func:`append_pages`);
    returns [B, L, Hq, 128].  Hq is a multiple of the pools' heads H; query head h reads key head
    ``h // (Hq // H)``.

    The prefix is ``prefix_tokens`` tokens in ``prefix_pages`` (int32 on the GPU), pages of the same
    pools or of ``prefix_pools = (kpool, vpool, page_tokens)``; every row sees all of it, and its keys
    are read once for the whole batch.  Of its own tokens row t of a sequence sees the first
    ``lengths[b] - new_lens[b] + t + 1`` (``causal``) or all ``lengths[b]``.  Rows that are no new
    tokens, and rows that see no key at all, come back as zeros.  ``out`` may be ``q`` itself, and must
    not otherwise share memory with an input.  No gradient is recorded."""
    check_heads("q", q, _HALVES)
    b, l, hq, _ = q.shape
    n_pages, h = _check_pools("", kpool, vpool, page_tokens, q.dtype)
    if h == 0 or hq == 0 or hq % h:
        raise ValueError(f"q has {hq} heads, which is no multiple of the pools' {h}")
    prefix_tokens = int(prefix_tokens)
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"softmax_scale must be positive and finite, got {scale}")
    d = _lib.AttendSharedDesc(batch=b, rows=l, q_heads=hq, kv_heads=h, causal=bool(causal), softmax_scale=scale,
                              prefix_tokens=prefix_tokens)
    _set_pages(d, kpool, vpool, n_pages, page_tokens, tables, lengths, new_lens, b)
    pk, pv = kpool, vpool
    if prefix_tokens:
        n, t = n_pages, page_tokens
        if prefix_pools is not None:
            pk, pv, t = prefix_pools
            n, ph = _check_pools("prefix ", pk, pv, t, q.dtype)
            if ph != h:
                raise ValueError(f"prefix pools have {ph} heads, the sequences' {h}")
        if prefix_pages is None:
            raise ValueError("prefix_tokens without prefix_pages")
        if prefix_tokens < 0 or prefix_tokens > prefix_pages.numel() * t:
            raise ValueError(f"{prefix_tokens} prefix tokens do not lie in {prefix_pages.numel()} pages of {t}")
        _int32_vector("prefix_pages", prefix_pages, prefix_pages.numel())
        d.prefix_k_pool, d.prefix_v_pool = pk.data_ptr(), pv.data_ptr()
        d.prefix_n_pages, d.prefix_page_tokens, d.prefix_pages = n, t, prefix_pages.data_ptr()
    else:
        prefix_pages = None
    if out is None:
        out = empty_as(q)
    else:
        _check_out(out, q)
    d.q, d.out = q.data_ptr(), out.data_ptr()
    d.q_sb, d.q_st, d.q_sh = strides("q", q)
    d.out_sb, d.out_st, d.out_sh = strides("out", out)
    same_device(("k_pool", "v_pool", "q", "out", "tables", "lengths", "new_lens", "prefix_pages",
                 "prefix k_pool", "prefix v_pool"),
                (kpool, vpool, q, out, tables, lengths, new_lens, prefix_pages, pk, pv))
    if q.numel() == 0:
        return out
    size = ctypes.c_int64(0)
    status = _lib.load().skv_attend_shared_workspace(ctypes.byref(d), ctypes.byref(size))
    if status:
        _lib.check("skv_attend_shared_workspace", status)
    ws = None
    if size.value:
        # a block of this call's own: two graphs captured on one stream may replay side by side
        ws = torch.empty(size.value, dtype=torch.uint8, device=q.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), size.value
    launch("skv_attend_shared", d, q.device)
    del ws
    return out


def history_pages(cache: SlotKVCache) -> tuple[torch.Tensor, int, tuple[torch.Tensor, torch.Tensor, int]]:
    """(prefix pages, prefix tokens, prefix pools) of a committed frame-slot cache with a batch of
    one, for :func:`attend_shared`: its frames, sink and window in order, as the history that a batch
    of rollouts goes on from.  The cache must hold rotated keys (allocated without ``rope=``) in
    bfloat16 or float16, and must not be committed to again while the rollouts read it."""
    g = cache.geom
    if g.batch != 1:
        raise ValueError(f"a shared history has a batch of one, this cache has {g.batch}")
    if cache.rope is not None:
        raise ValueError("a shared history needs rotated keys: this cache rotates them on load (rope=)")
    if cache.dtype not in _HALVES:
        raise ValueError(f"a shared history needs a bfloat16 or float16 cache, got {cache.dtype}")
    frames = cache.local_end // g.frame_tokens
    pages = torch.tensor(cache.table[:frames], dtype=torch.int32).to(cache.device)
    return pages, cache.local_end, (cache.kpool, cache.vpool, g.frame_tokens)
