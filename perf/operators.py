"""The operators of sequences that share a history, as timed cases over their public entry points.

* ``norm_rope``  RMS norm of every query and key head with the position rotation in the same pass
                 (``qk_norm_rope``); with ``train`` the backward pass as well;
* ``append``     new keys and values into a paged cache, keys normalised and rotated on the way and
                 the queries with them (``append_pages``);
* ``shared``     attention of a batch whose sequences share a long prefix and go on in pages of
                 their own (``attend_shared``).

Pages are frame slots with a batch of one (K ``[pages, 1, H, Tp, 128]``, V transposed), so a page
holds ``page`` tokens and ``Tp`` is that number rounded up to 64.  ``run`` computes the plain forms
with elementary tensor operations in float32, rounded once at the end; with ``own`` it makes a
user's calls of the framework.
"""

from __future__ import annotations

import math
from typing import Any

import torch

own = False

D = 128
DEVICE = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
PAGES = (16, 48, 64, 100, 128, 256, 390, 880, 1560)


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _norm_rope(**kw: Any) -> dict:
    return dict(dict(kind="norm_rope", dtype="bf16", batch=1, rot=128, interleaved=False, packed=False,
                     train=False), **kw)


def _append(**kw: Any) -> dict:
    return dict(dict(kind="append", dtype="bf16", rot=128, interleaved=False, ragged=False), **kw)


def _shared(**kw: Any) -> dict:
    return dict(dict(kind="shared", dtype="bf16", length=1, causal=True, ragged=False), **kw)


def listed() -> list[dict]:
    return [
        # a few tokens of one stream, q and k as slices of one projection: the smallest call
        _norm_rope(name="norm_rope_few", length=16, q_heads=12, k_heads=12, packed=True),
        # a chunk of three 1560-token frames of a 40-head model, rotate-half on 96 channels
        _norm_rope(name="norm_rope_chunk", length=4680, q_heads=40, k_heads=40, rot=96),
        # training on two 8190-token clips of a 24-head model, rotation of neighbouring channels
        _norm_rope(name="norm_rope_train", batch=2, length=8190, q_heads=24, k_heads=24,
                   interleaved=True, train=True),
        # a float32 fine-tuning step with shared key heads, partial rotation and an odd length
        _norm_rope(name="norm_rope_train_f32", dtype="f32", batch=3, length=777, q_heads=16, k_heads=4,
                   rot=64, packed=True, train=True),
        # the next token of one sequence: the smallest append
        _append(name="append_token", batch=1, length=1, q_heads=12, kv_heads=12, past=700, prefix=390, page=64),
        # the next token of a batch in float16 with shared key heads
        _append(name="append_batch", dtype="f16", batch=64, length=1, q_heads=32, kv_heads=8, past=2000,
                prefix=8190, page=64),
        # frames of eight rollouts, padded to the longest, in pages of one 1560-token frame
        _append(name="append_frames", batch=8, length=1560, q_heads=24, kv_heads=24, past=1560,
                prefix=32760, page=1560, interleaved=True, ragged=True),
        # one token after one 390-token frame: the smallest attention
        _shared(name="shared_token", batch=1, q_heads=12, kv_heads=12, prefix=390, own=64, page=64),
        # the next token of 32 sequences after a window of 21 frames
        _shared(name="shared_decode", batch=32, q_heads=32, kv_heads=8, prefix=32760, own=1560, page=64),
        # four rollouts of a 12-head model, each attending a whole 390-token frame in frame pages
        _shared(name="shared_frames", batch=4, length=390, q_heads=12, kv_heads=12, prefix=8190, own=1170,
                page=390, causal=False),
        # a few drafted tokens for each of 24 sequences, padded, float16, odd lengths and pages
        _shared(name="shared_drafts", dtype="f16", batch=24, length=5, q_heads=24, kv_heads=8, prefix=4097,
                own=777, page=48, ragged=True),
        # the next token of a large batch after a very long prefix: the largest
        _shared(name="shared_large", batch=128, q_heads=64, kv_heads=8, prefix=131072, own=4096, page=64),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _heads(rng) -> tuple[int, int]:
    kv = rng.choice((1, 2, 3, 4, 5, 8, 12, 16, 24, 40))
    return kv * rng.choice((1, 1, 2, 3, 4, 5, 8) if kv <= 8 else (1, 1, 2)), kv


def draw(rng) -> dict:
    kind = rng.choice(("norm_rope", "append", "shared", "shared"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    rot, inter = rng.choice((32, 64, 96, 128, 128)), rng.random() < 0.5
    q_heads, kv_heads = _heads(rng)
    if kind == "norm_rope":
        batch = _log(rng, 1, 16)
        return _norm_rope(dtype=rng.choice(("bf16", "bf16", "f16", "f32")), batch=batch,
                          length=_log(rng, 1, max(1, 650_000 // (batch * (q_heads + kv_heads)))),
                          q_heads=q_heads, k_heads=kv_heads, rot=rot, interleaved=inter,
                          packed=rng.random() < 0.5, train=rng.random() < 0.6)
    page = rng.choice(PAGES)
    if kind == "append":
        batch = _log(rng, 1, 128)
        length = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 200_000 // (batch * (q_heads + 2 * kv_heads))))
        past = _log(rng, 1, max(1, min(2048, 1_000_000 // (batch * kv_heads))))
        return _append(dtype=dtype, batch=batch, length=length, q_heads=q_heads, kv_heads=kv_heads, past=past,
                       prefix=rng.choice((0, _log(rng, 1, 60000))), page=page, rot=rot, interleaved=inter,
                       ragged=length > 1 and rng.random() < 0.5)
    batch = _log(rng, 1, 128)
    length = 1 if rng.random() < 0.5 else _log(rng, 2, 400)
    length = min(length, max(1, 8192 // batch))
    rows = batch * length * q_heads
    prefix = _log(rng, 1, max(1, min(131072, 500_000_000 // rows, 1_000_000 // kv_heads)))
    past = _log(rng, 1, max(1, min(4096, 100_000_000 // rows, 4_000_000 // (batch * kv_heads))))
    return _shared(dtype=dtype, batch=batch, length=length, q_heads=q_heads, kv_heads=kv_heads,
                   prefix=0 if rng.random() < 0.1 else prefix, own=past + length, page=page,
                   causal=rng.random() < 0.7, ragged=length > 1 and rng.random() < 0.5)


def work(case: dict) -> dict:
    e, b, n = SIZES[case["dtype"]], case["batch"], case["length"]
    if case["kind"] == "norm_rope":
        x = b * n * (case["q_heads"] + case["k_heads"]) * D
        tables = n * case["rot"] * 4
        if not case["train"]:
            return {"bytes": 2 * e * x + tables, "flops": 8 * x}
        return {"bytes": 5 * e * x + 2 * tables, "flops": 28 * x}
    tokens = b * n * (0.5 if case["ragged"] else 1.0)
    if case["kind"] == "append":
        x = tokens * (case["q_heads"] + 2 * case["kv_heads"]) * D
        return {"bytes": 2 * e * x, "flops": 8 * tokens * (case["q_heads"] + case["kv_heads"]) * D}
    keys = (case["own"] + n) / 2
    kv = (case["prefix"] + b * keys) * case["kv_heads"] * 2 * D * e
    return {"bytes": kv + 2 * tokens * case["q_heads"] * D * e,
            "flops": 4 * D * tokens * case["q_heads"] * (case["prefix"] + keys)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _tables(rows: int, rot: int) -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin float32 [rows, rot / 2] of position * 10000^(-2i / rot), from float64 angles."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    ang = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEVICE), inv)
    return ang.cos().float(), ang.sin().float()


def _projection(g, shape, dtype):
    """Rows of a projection: each token has a magnitude of its own."""
    size = torch.exp(0.5 * torch.randn(*shape[:2], 1, 1, generator=g, device=DEVICE))
    return (torch.randn(shape, generator=g, device=DEVICE) * size).to(dtype)


def _weight(g):
    return 1.0 + 0.2 * torch.randn(D, generator=g, device=DEVICE)


def _pools(g, n_pages, heads, page, dtype):
    """K and V pools with tokens in every page; the padding behind a page's tokens is zero."""
    padded = (page + 63) // 64 * 64
    kpool = torch.randn(n_pages, 1, heads, padded, D, generator=g, device=DEVICE, dtype=dtype)
    vpool = torch.randn(n_pages, 1, heads, D, padded, generator=g, device=DEVICE, dtype=dtype)
    kpool[:, :, :, page:] = 0
    vpool[..., page:] = 0
    return kpool, vpool


def _lengths(g, case, most):
    """(tokens of each sequence with the new ones, new tokens of each or None), int32."""
    b, n = case["batch"], case["length"]
    new = None
    if case["ragged"]:
        new = torch.randint(0, n + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
        new[0] = n
    past = torch.randint(0, most + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
    return past + (n if new is None else new), new


def _page_tables(g, n_own, batch, n_prefix):
    """Tables of ``n_own`` pages for each sequence and the prefix's list, out of one shuffled pool."""
    order = torch.randperm(batch * n_own + n_prefix, generator=g, device=DEVICE).to(torch.int32)
    return order[: batch * n_own].reshape(batch, n_own).contiguous(), order[batch * n_own:].contiguous()


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, b, n = DTYPES[case["dtype"]], case["batch"], case["length"]
    hq = case["q_heads"]
    s: dict[str, Any] = {"case": case}
    if case["kind"] == "norm_rope":
        hk = case["k_heads"]
        if case["packed"]:
            x = _projection(g, (b, n, hq + 2 * hk, D), dtype)
            s["q"], s["k"] = x[:, :, :hq], x[:, :, hq:hq + hk]
        else:
            s["q"], s["k"] = _projection(g, (b, n, hq, D), dtype), _projection(g, (b, n, hk, D), dtype)
        s["wq"], s["wk"] = _weight(g), _weight(g)
        s["cos"], s["sin"] = _tables(n, case["rot"])
        if case["train"]:
            s["gq"] = torch.randn(b, n, hq, D, generator=g, device=DEVICE, dtype=dtype)
            s["gk"] = torch.randn(b, n, hk, D, generator=g, device=DEVICE, dtype=dtype)
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_()
        return s
    hkv, page = case["kv_heads"], case["page"]
    if case["kind"] == "append":
        s["q"], s["k"] = _projection(g, (b, n, hq, D), dtype), _projection(g, (b, n, hkv, D), dtype)
        s["v"] = torch.randn(b, n, hkv, D, generator=g, device=DEVICE, dtype=dtype)
        s["wq"], s["wk"] = _weight(g), _weight(g)
        s["cos"], s["sin"] = _tables(case["prefix"] + case["past"] + n, case["rot"])
        n_own = -(-(case["past"] + n) // page)
        s["tables"], _ = _page_tables(g, n_own, b, 0)
        s["kpool"], s["vpool"] = _pools(g, b * n_own, hkv, page, dtype)
        s["lengths"], s["new"] = _lengths(g, case, case["past"])
        return s
    n_own, n_prefix = -(-case["own"] // page), -(-case["prefix"] // page)
    s["q"] = (1.5 * torch.randn(b, n, hq, D, generator=g, device=DEVICE)).to(dtype)
    s["tables"], s["prefix_pages"] = _page_tables(g, n_own, b, n_prefix)
    s["kpool"], s["vpool"] = _pools(g, b * n_own + n_prefix, hkv, page, dtype)
    s["lengths"], s["new"] = _lengths(g, case, case["own"] - n)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _plain_norm_rope(x, weight, cos, sin, interleaved):
    """float32 of ``x`` normalised over its channels, weighted, and rotated by tables that broadcast."""
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    half = cos.shape[-1]
    a, b = ((y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if interleaved
            else (y[..., :half], y[..., half:2 * half]))
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _plain_train(s):
    case = s["case"]
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    q = _plain_norm_rope(s["q"], s["wq"], cos, sin, case["interleaved"]).to(s["q"].dtype)
    k = _plain_norm_rope(s["k"], s["wk"], cos, sin, case["interleaved"]).to(s["k"].dtype)
    if not case["train"]:
        return q, k
    return (q.detach(), k.detach(),
            *torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"])))


def _new_tokens(s):
    """(new tokens [B, 1], own index of every row [B, L], whether the row is a token [B, L])."""
    n = s["case"]["length"]
    row = torch.arange(n, device=DEVICE)[None]
    new = (torch.full_like(s["lengths"], n) if s["new"] is None else s["new"])[:, None]
    return new, s["lengths"][:, None] - new + row, row < new


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    _, at, there = _new_tokens(s)
    where = at.clamp(min=0)
    cos, sin = (t[(case["prefix"] + where).clamp(max=t.shape[0] - 1)][:, :, None] for t in (s["cos"], s["sin"]))
    q = _plain_norm_rope(s["q"], s["wq"], cos, sin, case["interleaved"])
    k = _plain_norm_rope(s["k"], s["wk"], cos, sin, case["interleaved"])
    q = torch.where(there[:, :, None, None], q, 0.0).to(s["q"].dtype)
    pages = s["tables"].gather(1, (where // page).clamp(max=s["tables"].shape[1] - 1).long()).long()
    offset, k, v = (where % page).long(), k.to(s["kpool"].dtype), s["v"]
    if s["new"] is not None:
        pages, offset, k, v = (t[there] for t in (pages, offset, k, v))
    s["kpool"][pages, 0, :, offset] = k
    s["vpool"][pages, 0, :, :, offset] = v
    return q, s["kpool"], s["vpool"]


def _plain_shared(s):
    """Scores of the prefix (one product for the whole batch) and of each sequence's own pages,
    one softmax over both, and their weighted values."""
    case = s["case"]
    b, n, hq, _ = s["q"].shape
    hkv, page = case["kv_heads"], case["page"]
    group = hq // hkv
    q = s["q"].float().reshape(b, n, hkv, group, D) * D ** -0.5
    prefix = s["prefix_pages"].long()
    kp = s["kpool"][prefix, 0, :, :page].float().transpose(0, 1).reshape(hkv, -1, D)[:, : case["prefix"]]
    vp = s["vpool"][prefix, 0, :, :, :page].float().permute(1, 0, 3, 2).reshape(hkv, -1, D)[:, : case["prefix"]]
    own_pages = s["tables"].long()
    ko = s["kpool"][own_pages, 0, :, :page].float().transpose(1, 2).reshape(b, hkv, -1, D)
    vo = s["vpool"][own_pages, 0, :, :, :page].float().permute(0, 2, 1, 4, 3).reshape(b, hkv, -1, D)
    qp = q.permute(2, 0, 1, 3, 4).reshape(hkv, b * n * group, D)
    sp = (qp @ kp.transpose(1, 2).contiguous()).reshape(hkv, b, n * group, -1).transpose(0, 1)
    qo = q.permute(0, 2, 1, 3, 4).reshape(b, hkv, n * group, D)
    so = qo @ ko.transpose(2, 3).contiguous()
    _, at, there = _new_tokens(s)
    last = at if case["causal"] else (s["lengths"][:, None] - 1).expand(b, n)
    key = torch.arange(so.shape[-1], device=DEVICE)
    seen = (key[None, None] <= last[:, :, None]) & (key[None, None] < s["lengths"][:, None, None])
    seen = seen.repeat_interleave(group, 1)[:, None]  # [B, 1, L * group, keys]
    so = so.masked_fill(~seen, -math.inf)
    vo = vo * (key < s["lengths"][:, None])[:, None, :, None]
    top = so.amax(-1, keepdim=True)
    if case["prefix"]:
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    po = torch.exp(so - top)
    pp = torch.exp(sp - top)
    total = po.sum(-1, keepdim=True) + pp.sum(-1, keepdim=True)
    out = po @ vo
    out = out + (pp.transpose(0, 1).reshape(hkv, b * n * group, -1) @ vp).reshape(hkv, b, n * group, D).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0).reshape(b, hkv, n, group, D)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, n, hq, D)
    return torch.where(there[:, :, None, None], out, 0.0).to(s["q"].dtype)


def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if own:
        from solarwm_amd import append_pages, attend_shared, qk_norm_rope

        if kind == "norm_rope":
            q, k = qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], norm_q=(s["wq"], EPS), norm_k=(s["wk"], EPS),
                                interleaved=case["interleaved"])
            if not case["train"]:
                return q, k
            return (q.detach(), k.detach(),
                    *torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"])))
        if kind == "append":
            q = append_pages(s["k"], s["v"], s["kpool"], s["vpool"], s["tables"], s["lengths"],
                             page_tokens=case["page"], new_lens=s["new"], q=s["q"], cos=s["cos"], sin=s["sin"],
                             position0=case["prefix"], interleaved=case["interleaved"],
                             norm_q=(s["wq"], EPS), norm_k=(s["wk"], EPS))
            return q, s["kpool"], s["vpool"]
        return attend_shared(s["q"], s["kpool"], s["vpool"], s["tables"], s["lengths"], page_tokens=case["page"],
                             prefix_pages=s["prefix_pages"], prefix_tokens=case["prefix"], new_lens=s["new"],
                             causal=case["causal"])
    if kind == "norm_rope":
        return _plain_train(s)
    return _plain_append(s) if kind == "append" else _plain_shared(s)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _pairs(rot, interleaved):
    i = torch.arange(rot // 2, device=DEVICE)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def _exact_heads(x, w, cos, sin, rot, interleaved, grad=None):
    """norm and rotation of x [..., H, 128] in float64; with ``grad`` also (dx, dw)."""
    x, w, cos, sin = x.detach().double(), w.detach().double(), cos.double(), sin.double()
    r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
    y = w * (x * r)
    i, j = _pairs(rot, interleaved)
    z = y.clone()
    z[..., i] = y[..., i] * cos - y[..., j] * sin
    z[..., j] = y[..., i] * sin + y[..., j] * cos
    if grad is None:
        return z
    g = grad.double()
    gy = g.clone()
    gy[..., i] = g[..., i] * cos + g[..., j] * sin
    gy[..., j] = g[..., j] * cos - g[..., i] * sin
    dw = (gy * x * r).flatten(0, -2).sum(0)
    u = gy * w
    return z, r * u - x * r ** 3 * (u * x).sum(-1, keepdim=True) / D, dw


def _exact_shared(s):
    case = s["case"]
    b, n, hq, _ = s["q"].shape
    hkv, page = case["kv_heads"], case["page"]
    group = hq // hkv
    out = torch.zeros(b, n, hq, D, dtype=torch.float64, device=DEVICE)
    lengths = s["lengths"].tolist()
    new = [n] * b if s["new"] is None else s["new"].tolist()
    prefix, tables = s["prefix_pages"].long(), s["tables"].long()
    for h in range(hkv):
        heads = slice(h * group, (h + 1) * group)
        kp = s["kpool"][prefix, 0, h, :page].reshape(-1, D)[: case["prefix"]].double()
        vp = s["vpool"][prefix, 0, h, :, :page].transpose(1, 2).reshape(-1, D)[: case["prefix"]].double()
        for i in range(b):
            if not new[i]:
                continue
            ko = s["kpool"][tables[i], 0, h, :page].reshape(-1, D)[: lengths[i]].double()
            vo = s["vpool"][tables[i], 0, h, :, :page].transpose(1, 2).reshape(-1, D)[: lengths[i]].double()
            q = s["q"][i, : new[i], heads].double().reshape(-1, D)
            score = torch.cat((q @ kp.T, q @ ko.T), 1) / math.sqrt(D)
            if case["causal"]:
                last = case["prefix"] + lengths[i] - new[i] + torch.arange(new[i], device=DEVICE)
                hidden = torch.arange(score.shape[1], device=DEVICE)[None] > last.repeat_interleave(group)[:, None]
                score[hidden] = -math.inf
            p = torch.softmax(score, 1)
            out[i, : new[i], heads] = (p[:, : case["prefix"]] @ vp + p[:, case["prefix"]:] @ vo).reshape(-1, group, D)
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "norm_rope":
        cos, sin = s["cos"][:, None], s["sin"][:, None]
        args = (cos, sin, case["rot"], case["interleaved"])
        if not case["train"]:
            return _exact_heads(s["q"], s["wq"], *args), _exact_heads(s["k"], s["wk"], *args)
        q, dq, dwq = _exact_heads(s["q"], s["wq"], *args, s["gq"])
        k, dk, dwk = _exact_heads(s["k"], s["wk"], *args, s["gk"])
        return q, k, dq, dk, dwq, dwk
    if case["kind"] == "shared":
        return _exact_shared(s)
    n, page = case["length"], case["page"]
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    kpool, vpool = s["kpool"].double(), s["vpool"].double()
    new = [n] * case["batch"] if s["new"] is None else s["new"].tolist()
    for i, (length, m) in enumerate(zip(s["lengths"].tolist(), new)):
        at = torch.arange(length - m, length, device=DEVICE)
        tables = (s["cos"][case["prefix"] + at][:, None], s["sin"][case["prefix"] + at][:, None])
        q[i, :m] = _exact_heads(s["q"][i, :m], s["wq"], *tables, case["rot"], case["interleaved"])
        k = _exact_heads(s["k"][i, :m], s["wk"], *tables, case["rot"], case["interleaved"])
        pages, offset = s["tables"][i].long()[at // page], at % page
        kpool[pages, 0, :, offset] = k
        vpool[pages, 0, :, :, offset] = s["v"][i, :m].double()
    return q, kpool, vpool
