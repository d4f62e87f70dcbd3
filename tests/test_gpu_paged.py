"""Paged append and shared-prefix attention against float64.

Append: V bit for bit, K and q within the bar of test_gpu_qknorm (one rounding plus 16 fp32
roundings of the pair's values), everything else of the pools untouched.

Attention, per element of the output, with A = sum_j p_j |v_j| over the row's keys:
  * the probabilities are rounded to the pool's type for the matrix product: half a step of A;
  * the output is rounded once: half a step of its value;
  * float16 only: probabilities below 2^-14 of a maximum that is at least 1 step by 2^-24, half of
    that for each key times its |v|;
  * fp32: a score is 128 products with sums (160 roundings of the sum of absolute products S, which
    move p and its sum by that much each), exp2 and the sums of l and of the output (64 + a 64th of
    the keys, on A).
"""

import math

import pytest
import torch

from solarwm_amd import (append_pages, apply_cache_updates, attend_cached, attend_shared, history_pages,
                         kernels, make_kv_cache_allocator, qk_norm_rope)

from .test_gpu_qknorm import EPS, HALF, TINY, U, _near, _reference, _rows, _tables, _weight

pytestmark = pytest.mark.gpu

D = 128
BF, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _pools(n_pages, heads, page, dtype, dev, seed):
    """Pools whose every element is set; the padding behind a page's tokens holds NaN."""
    tp = kernels.padded_tokens(page)
    k = torch.randn(n_pages, 1, heads, tp, D, generator=_gen(seed)).to(dtype)
    v = torch.randn(n_pages, 1, heads, D, tp, generator=_gen(seed + 1)).to(dtype)
    k[:, :, :, page:] = float("nan")
    v[..., page:] = float("nan")
    return k.to(dev), v.to(dev)


def _places(tables, lengths, new, rows, page, n_pages):
    """[(sequence, row, page, offset)] of the tokens that have a place, and the rows that are tokens."""
    places, there = [], torch.zeros(len(lengths), rows, dtype=torch.bool)
    for b, length in enumerate(lengths):
        n = rows if new is None else min(max(new[b], 0), rows)
        for t in range(n):
            there[b, t] = True
            own = length - n + t
            if own < 0 or own // page >= tables.shape[1]:
                continue
            p = int(tables[b, own // page])
            if 0 <= p < n_pages:
                places.append((b, t, p, own % page))
    return places, there


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


APPENDS = [  # page, batch, rows, q heads, kv heads, rot, lengths with the new tokens, new_lens
    (64, 1, 1, 4, 4, 128, [1], None),
    (64, 3, 1, 8, 2, 64, [64, 65, 200], None),
    (16, 2, 5, 3, 3, 96, [5, 37], None),
    (48, 3, 7, 10, 5, 16, [48, 51, 3], [7, 0, 3]),
    (64, 2, 9, 2, 1, 128, [9, 73], [9, 4]),
    (100, 3, 130, 6, 2, 64, [130, 333, 90], [130, 77, 8]),
    (390, 2, 400, 1, 1, 112, [1000, 401], None),
    (1, 2, 20, 2, 2, 32, [25, 20], None),
]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("case", APPENDS)
def test_append(gpu, case, inter, dtype):
    page, b, n, hq, hkv, rot, lengths, new = case
    print("append_pages", case, inter, dtype, flush=True)
    width = -(-max(lengths) // page)
    n_pages = b * width + 3
    kpool, vpool = _pools(n_pages, hkv, page, dtype, gpu, 1)
    k0, v0 = kpool.cpu(), vpool.cpu()
    tables = torch.randperm(n_pages, generator=_gen(3))[: b * width].reshape(b, width).int()
    q, k, v = (_rows((b, n, h, D), 4 + i, dtype, gpu) for i, h in enumerate((hq, hkv, hkv)))
    wq, wk = _weight(7, torch.float32, gpu), _weight(8, dtype, gpu)
    p0 = 11
    cos, sin = _tables(p0 + max(lengths), rot, gpu)
    got = append_pages(k, v, kpool, vpool, tables.to(gpu), _i32(lengths, gpu), page_tokens=page,
                       new_lens=None if new is None else _i32(new, gpu), q=q, cos=cos, sin=sin,
                       position0=p0, interleaved=inter, norm_q=(wq, EPS), norm_k=(wk, EPS))
    places, there = _places(tables, lengths, new, n, page, n_pages)
    own = torch.tensor([[length - (n if new is None else new[i]) + t for t in range(n)]
                        for i, length in enumerate(lengths)]).clamp(0, max(lengths) - 1)
    c, s = (t.cpu().double()[p0 + own][:, :, None] for t in (cos, sin))
    zq, sq = _reference(q, wq, c, s, rot, inter, True)
    zk, sk = _reference(k, wk, c, s, rot, inter, True)
    _near("q", got.cpu()[there], zq[there], sq[there], dtype, 16)
    assert torch.equal(got.cpu()[~there], torch.zeros_like(got.cpu()[~there]))
    kc, vc, vin = kpool.cpu(), vpool.cpu(), v.cpu()
    for i, t, p, o in places:
        _near("k", kc[p, 0, :, o], zk[i, t], sk[i, t], dtype, 16)
        assert torch.equal(vc[p, 0, :, :, o], vin[i, t])
        k0[p, 0, :, o], v0[p, 0, :, :, o] = kc[p, 0, :, o], vin[i, t]
    assert torch.equal(kc.view(torch.int16), k0.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), v0.view(torch.int16))


@pytest.mark.parametrize("rows", [1, 12])
def test_append_tokens_without_a_place(gpu, rows):
    """Entries outside the pool, tokens behind the table, lengths below the new tokens and new_lens
    beyond the rows write what has a place and nothing else."""
    page, hkv, n_pages = 16, 3, 6
    kpool, vpool = _pools(n_pages, hkv, page, BF, gpu, 21)
    k0, v0 = kpool.cpu(), vpool.cpu()
    tables = torch.tensor([[-1, 4], [5, n_pages], [0, 1], [2, 3], [2**31 - 1, -2**31]], dtype=torch.int32)
    lengths = [16, 18, 40, rows - 1, 20]
    new = [rows, rows, rows, rows + 5, 0]
    k, v = _rows((5, rows, hkv, D), 22, BF, gpu), _rows((5, rows, hkv, D), 23, BF, gpu)
    assert append_pages(k, v, kpool, vpool, tables.to(gpu), _i32(lengths, gpu), page_tokens=page,
                        new_lens=_i32(new, gpu)) is None
    places, _ = _places(tables, lengths, new, rows, page, n_pages)
    for i, t, p, o in places:
        k0[p, 0, :, o], v0[p, 0, :, :, o] = k[i, t].cpu(), v[i, t].cpu()
    assert torch.equal(kpool.cpu().view(torch.int16), k0.view(torch.int16))
    assert torch.equal(vpool.cpu().view(torch.int16), v0.view(torch.int16))


def test_append_given_positions(gpu):
    """Positions per token replace the token's own index; q in place; a position outside the table
    makes NaN of the rotated channels of that token alone."""
    page, b, n = 64, 2, 3
    kpool, vpool = _pools(4, 2, page, BF, gpu, 31)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=gpu)
    q, k, v = (_rows((b, n, 2, D), 32 + i, BF, gpu) for i in range(3))
    cos, sin = _tables(30, 64, gpu)
    pos = torch.tensor([[3, 17, 29], [0, 30, 5]])
    want_q, want_k = qk_norm_rope(q, k, cos, sin, norm_q=(None, EPS), norm_k=(None, EPS), positions=pos.to(gpu))
    packed = torch.stack((q, q))
    out = append_pages(k, v, kpool, vpool, tables, _i32([66, 3], gpu), page_tokens=page, q=packed[1],
                       out=packed[1], cos=cos, sin=sin, positions=pos.int().to(gpu) - 4, position0=4,
                       norm_q=(None, EPS), norm_k=(None, EPS))
    assert out.data_ptr() == packed[1].data_ptr()
    assert torch.equal(out.view(torch.int16), want_q.view(torch.int16)) and torch.equal(packed[0], q)
    assert torch.isnan(out[1, 1][..., :64]).all() and not torch.isnan(out[1, 1][..., 64:]).any()
    got = torch.stack([torch.stack([kpool[0, 0, :, 63], kpool[1, 0, :, 0], kpool[1, 0, :, 1]]),
                       kpool[2, 0, :, :3].transpose(0, 1)])
    assert torch.equal(got.view(torch.int16), want_k.view(torch.int16))


# ---------------------------------------------------------------------------------------------
def _gather(kpool, vpool, page, ids, tokens):
    """float64 K, V [tokens, H, D] of a page list and which tokens are there."""
    n_pages, _, h = kpool.shape[:3]
    k = torch.zeros(tokens, h, D, dtype=torch.float64)
    v = torch.zeros(tokens, h, D, dtype=torch.float64)
    there = torch.zeros(tokens, dtype=torch.bool)
    for i in range(tokens):
        if i // page < len(ids) and 0 <= ids[i // page] < n_pages:
            k[i] = kpool[ids[i // page], 0, :, i % page].double()
            v[i] = vpool[ids[i // page], 0, :, :, i % page].double()
            there[i] = True
    return k, v, there


def _attention(q, own, lengths, new, causal, prefix=None, scale=D ** -0.5):
    """(want, bar) float64 [B, L, Hq, D]; own = (kpool, vpool, page, tables), prefix = (kpool, vpool,
    page, ids, tokens), all on the CPU."""
    dtype = q.dtype
    q = q.double()
    b, n, hq, _ = q.shape
    want, bar = torch.zeros_like(q), torch.zeros_like(q)
    kpool, vpool, page, tables = own
    hkv = kpool.shape[2]
    group = hq // hkv
    if prefix is not None:
        kp, vp, tp = _gather(*prefix)
    for i in range(b):
        m = n if new is None else min(max(new[i], 0), n)
        length = min(max(lengths[i], 0), tables.shape[1] * page)
        ko, vo, to = _gather(kpool, vpool, page, tables[i].tolist(), length)
        own0 = 0
        if prefix is not None:
            own0, ko, vo, to = kp.shape[0], torch.cat((kp, ko)), torch.cat((vp, vo)), torch.cat((tp, to))
        for t in range(m):
            seen = to.clone()
            if causal:
                seen[own0 + max(lengths[i] - m + t + 1, 0):] = False
            if not seen.any():
                continue
            for h in range(hkv):
                ks, vs = ko[seen, h], vo[seen, h]
                qs = q[i, t, h * group:(h + 1) * group]
                s = qs @ ks.T * scale
                p = torch.softmax(s, -1)
                o, a = p @ vs, p @ vs.abs()
                size = (qs.abs() @ ks.abs().T * scale).amax(-1, keepdim=True)
                rows = slice(h * group, (h + 1) * group)
                want[i, t, rows] = o
                e = HALF[dtype] * (a + o.abs()) * (1 + 2.0**-6) + TINY[dtype]
                if dtype == F16:
                    e = e + 2.0**-25 * vs.abs().sum(0)
                bar[i, t, rows] = e + U * (2 * 160 * size + 64 + ks.shape[0] / 64) * a
    return want, bar


def _check(got, want, bar, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bar).max()
    assert float(over) <= 0, (what, float(over), float((got - want).abs().max()), float(bar.max()))


ATTENDS = [  # batch, rows, q heads, kv heads, prefix, page, lengths, new_lens
    (1, 1, 1, 1, 0, 64, [1], None),
    (1, 1, 4, 4, 1, 64, [1], None),
    (1, 1, 12, 12, 390, 64, [64], None),
    (3, 1, 8, 2, 130, 64, [1, 64, 65], None),
    (2, 1, 5, 1, 1000, 16, [17, 0], [1, 0]),
    (5, 1, 32, 4, 64, 48, [100, 3, 47, 48, 49], None),  # 40 rows of a key head
    (20, 1, 16, 2, 257, 100, [7 * i for i in range(20)], [i % 3 != 0 for i in range(20)]),  # 160 rows
    (2, 5, 6, 2, 99, 48, [5, 60], None),
    (2, 9, 4, 2, 0, 100, [9, 130], [9, 2]),       # 18 rows of a sequence
    (3, 33, 2, 1, 70, 64, [33, 200, 40], [33, 20, 0]),
    (1, 150, 1, 1, 500, 390, [700], None),        # 150 rows of a sequence
    (2, 70, 3, 1, 0, 1, [70, 90], None),          # pages of one token
    (1, 1, 3, 1, 200, 64, [1500], None),          # a long sequence, split along its keys
    (1, 40, 2, 1, 0, 64, [1300], None),
]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", ATTENDS)
def test_attention(gpu, case, causal, dtype):
    b, n, hq, hkv, prefix, page, lengths, new = case
    print("attend_shared", case, causal, dtype, flush=True)
    new = None if new is None else [int(x) for x in new]
    width, n_pre = -(-max(lengths) // page) + 1, -(-prefix // page)
    n_pages = b * width + n_pre + 1
    kpool, vpool = _pools(n_pages, hkv, page, dtype, "cpu", 41)
    order = torch.randperm(n_pages, generator=_gen(43)).int()
    tables, ids = order[: b * width].reshape(b, width), order[b * width:b * width + n_pre]
    # what lies behind a sequence's tokens in its last page is no key, whatever it holds
    for i, length in enumerate(lengths):
        p, o = int(tables[i, length // page]), length % page
        kpool[p, 0, :, o:] = float("inf")
        vpool[p, 0, :, :, o:] = float("nan")
    q = (2 * torch.randn(b, n, hq, D, generator=_gen(44))).to(dtype)
    want, bar = _attention(q, (kpool, vpool, page, tables), lengths, new, causal,
                           (kpool, vpool, page, ids.tolist(), prefix) if prefix else None)
    got = attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables.to(gpu), _i32(lengths, gpu),
                        page_tokens=page, prefix_pages=ids.to(gpu), prefix_tokens=prefix,
                        new_lens=None if new is None else _i32(new, gpu), causal=causal)
    _check(got, want, bar)
    if new is not None:
        for i in range(b):
            assert not got[i, new[i]:].any()


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_pages_that_are_not_there(gpu, rows):
    """Missing pages of the prefix and of sequences, a table shorter than its sequence, a sequence
    with no page at all and no prefix tokens seen: zeros there, and no NaN elsewhere."""
    page, hkv, n_pages = 48, 2, 9
    kpool, vpool = _pools(n_pages, hkv, page, BF, "cpu", 51)
    tables = torch.tensor([[0, -1, 1], [n_pages, 2, 3], [-1, -1, -1], [4, 5, 6]], dtype=torch.int32)
    lengths = [130, 100, 140, 200]
    q = torch.randn(4, rows, 4, D, generator=_gen(52)).to(BF)
    for ids, prefix in (([7, -3, 8], 120), ([-1, 2**31 - 1], 96), ([], 0)):
        want, bar = _attention(q, (kpool, vpool, page, tables), lengths, None, True,
                               (kpool, vpool, page, ids, prefix) if prefix else None)
        got = attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables.to(gpu), _i32(lengths, gpu),
                            page_tokens=page, prefix_pages=_i32(ids, gpu), prefix_tokens=prefix)
        _check(got, want, bar, (ids, prefix))
        if not any(0 <= p < n_pages for p in ids):
            assert not got[2].any()
    empty = attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables[:, :0].to(gpu),
                          _i32([0] * 4, gpu), page_tokens=page)
    assert not empty.any()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("rows,hq", [(4, 2), (40, 1), (33, 4)])
def test_values_that_a_row_does_not_see(gpu, rows, hq, dtype):
    """Infinities and NaN in K and V of a token reach the rows that see it and no earlier ones."""
    page, at = 64, rows // 2
    kpool, vpool = _pools(3, 1, page, dtype, "cpu", 61)
    q = torch.randn(1, rows, hq, D, generator=_gen(62)).to(dtype)
    tables, length = torch.tensor([[1, 2]], dtype=torch.int32), 30 + rows
    want, bar = _attention(q, (kpool, vpool, page, tables), [length], None, True)

    def run():
        return attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables.to(gpu), _i32([length], gpu),
                             page_tokens=page).cpu()

    own = 30 + at
    p, o = int(tables[0, own // page]), own % page
    vpool[p, 0, 0, 5, o], vpool[p, 0, 0, 77, o] = float("inf"), float("nan")
    got = run()
    _check(got[:, :at], want[:, :at], bar[:, :at])
    assert torch.isinf(got[:, at:, :, 5]).all() and torch.isnan(got[:, at:, :, 77]).all()
    rest = [c for c in range(D) if c not in (5, 77)]
    _check(got[:, at:][..., rest], want[:, at:][..., rest], bar[:, at:][..., rest])
    vpool[p, 0, 0, 5, o] = vpool[p, 0, 0, 77, o] = 0
    kpool[p, 0, 0, o, 9] = float("nan")
    got = run()
    _check(got[:, :at], want[:, :at], bar[:, :at])
    assert torch.isnan(got[:, at:]).all()


@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_scores_far_apart(gpu, spread):
    """Scores that grow along the keys (every step raises the maximum by more than the running one
    may lag), shrink, or jump; the last key of the prefix outweighs all others."""
    page, hkv, prefix = 64, 1, 700
    kpool, vpool = _pools(16, hkv, page, BF, "cpu", 71)
    ids = list(range(11))
    q = torch.zeros(2, 1, 3, D)
    q[..., 0] = torch.tensor([1.0, -1.0, 0.25])[None, None]
    q = (q * math.sqrt(D)).to(BF)
    ramp = torch.arange(16 * page).reshape(16, page) / 16.0 * spread / 30.0
    kpool[:, 0, 0, :page, 0] = ramp.to(BF)
    kpool[10, 0, 0, 59, 0] = 40 * spread
    tables, lengths = torch.tensor([[11, 12], [13, 14]], dtype=torch.int32), [100, 65]
    want, bar = _attention(q, (kpool, vpool, page, tables), lengths, None, True, (kpool, vpool, page, ids, prefix))
    got = attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables.to(gpu), _i32(lengths, gpu),
                        page_tokens=page, prefix_pages=_i32(ids, gpu), prefix_tokens=prefix)
    _check(got, want, bar)


def test_strides_scale_and_other_pools(gpu):
    """q and out as slices, a scale, tables and lengths as slices, a prefix in pools of their own with
    other pages."""
    b, n, hq, hkv, page, ppage, prefix = 3, 2, 6, 3, 48, 100, 250
    kpool, vpool = _pools(8, hkv, page, BF, "cpu", 81)
    kpre, vpre = _pools(4, hkv, ppage, BF, "cpu", 83)
    tables = torch.tensor([[0, 1, 9], [2, 3, 9], [4, 5, 9]], dtype=torch.int32)
    lengths, ids = [50, 96, 2], [3, 0, 2]
    packed = torch.randn(b, n, hq + 2 * hkv, D, generator=_gen(85)).to(BF).to(gpu)
    out = torch.full((b, n, 2 * hq, D), 7.0, dtype=BF, device=gpu)
    want, bar = _attention(packed[:, :, :hq].cpu(), (kpool, vpool, page, tables[:, :2]), lengths, None, True,
                           (kpre, vpre, ppage, ids, prefix), scale=0.05)
    got = attend_shared(packed[:, :, :hq], kpool.to(gpu), vpool.to(gpu), tables.to(gpu)[:, :2],
                        _i32([9] + lengths, gpu)[1:], page_tokens=page, prefix_pages=_i32(ids, gpu),
                        prefix_tokens=prefix, prefix_pools=(kpre.to(gpu), vpre.to(gpu), ppage),
                        softmax_scale=0.05, out=out[:, :, ::2])
    _check(got, want, bar)
    assert got.data_ptr() == out.data_ptr() and (out[:, :, 1::2] == 7.0).all()


@pytest.mark.parametrize("b,n,hq,prefix", [(1, 1, 4, 100), (1, 3, 4, 5000), (3, 5, 6, 900), (2, 70, 2, 0), (40, 1, 8, 700)])
def test_out_is_q(gpu, b, n, hq, prefix):
    """Both operators write over their queries: the bits of a call with an output of its own."""
    hkv, page = 2, 64
    n_pre = -(-prefix // page)
    kpool, vpool = (t.to(gpu) for t in _pools(n_pre + 3 * b, hkv, page, BF, "cpu", 91))
    order = torch.randperm(n_pre + 3 * b, generator=_gen(92)).int().to(gpu)
    ids, tables = order[:n_pre].contiguous(), order[n_pre:].reshape(b, 3)
    lengths = torch.randint(n, 3 * page + 1, (b,), generator=_gen(93), dtype=torch.int32).to(gpu)
    q = torch.randn(b, n, hq, D, generator=_gen(94)).to(BF).to(gpu)
    k, v = (torch.randn(b, n, hkv, D, generator=_gen(95 + i)).to(BF).to(gpu) for i in range(2))
    angle = torch.rand(8192, 64, generator=_gen(97)).to(gpu)
    rope = dict(cos=angle.cos(), sin=angle.sin(), position0=prefix, norm_q=(None, 1e-6), norm_k=(None, 1e-6))

    def step(q, out):
        q = append_pages(k, v, kpool, vpool, tables, lengths, page_tokens=page, q=q, out=out, **rope)
        return attend_shared(q, kpool, vpool, tables, lengths, page_tokens=page, prefix_pages=ids,
                             prefix_tokens=prefix, out=out)

    want = step(q, None)
    got = step(q, q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


def test_many_splits_and_many_rows(gpu):
    """A long prefix split over the chip for few rows, and for many row blocks, against float64 on the
    GPU (float64 products of the same pools)."""
    hkv, page, prefix = 2, 64, 20000
    n_pre = -(-prefix // page)
    kpool, vpool = (t.to(gpu) for t in _pools(n_pre + 130, hkv, page, BF, "cpu", 91))
    ids = torch.randperm(n_pre, generator=_gen(93)).int().to(gpu)
    for b, hq in ((1, 2), (65, 16)):
        tables = torch.arange(n_pre, n_pre + 2 * b, dtype=torch.int32, device=gpu).reshape(b, 2)
        lengths = [1 + (37 * i) % 128 for i in range(b)]
        q = torch.randn(b, 1, hq, D, generator=_gen(94)).to(BF).to(gpu)
        got = attend_shared(q, kpool, vpool, tables, _i32(lengths, gpu), page_tokens=page,
                            prefix_pages=ids, prefix_tokens=prefix)
        kp = kpool[ids.long(), 0, :, :page].transpose(0, 1).reshape(hkv, -1, D)[:, :prefix].double()
        vp = vpool[ids.long(), 0, :, :, :page].permute(1, 0, 3, 2).reshape(hkv, -1, D)[:, :prefix].double()
        for i in range(b):
            for h in range(hkv):
                ko = kpool[tables[i].long(), 0, h, :page].reshape(-1, D)[: lengths[i]].double()
                vo = vpool[tables[i].long(), 0, h, :, :page].transpose(1, 2).reshape(-1, D)[: lengths[i]].double()
                ks, vs = torch.cat((kp[h], ko)), torch.cat((vp[h], vo))
                qs = q[i, 0, h * hq // hkv:(h + 1) * hq // hkv].double()
                p = torch.softmax(qs @ ks.T * D ** -0.5, -1)
                o, a = p @ vs, p @ vs.abs()
                size = (qs.abs() @ ks.abs().T * D ** -0.5).amax(-1, keepdim=True)
                bar = HALF[BF] * (a + o.abs()) * (1 + 2.0**-6) + U * (320 * size + 64 + ks.shape[0] / 64) * a
                err = (got[i, 0, h * hq // hkv:(h + 1) * hq // hkv].double() - o).abs() - bar
                assert float(err.max()) <= 0, (b, i, h, float(err.max()))


def _listed(kpool, vpool, page, ids, tokens):
    """float64 K, V [H, tokens, D] of a page list on the GPU, and which tokens are there."""
    at = ids.long().clamp(0, kpool.shape[0] - 1)
    h = kpool.shape[2]
    k = kpool[at, 0, :, :page].transpose(0, 1).reshape(h, -1, D)[:, :tokens].double()
    v = vpool[at, 0, :, :, :page].permute(1, 0, 3, 2).reshape(h, -1, D)[:, :tokens].double()
    there = ((ids >= 0) & (ids < kpool.shape[0])).repeat_interleave(page)[:tokens]
    return torch.where(there[:, None], k, 0.0), torch.where(there[:, None], v, 0.0), there


def _check_sequence(got, q, k, v, seen, dtype, what):
    """One sequence's rows [L, Hq, D] against float64 attention over the keys that ``seen`` [L, T] names."""
    n, hq, _ = q.shape
    h = k.shape[0]
    qs = q.double().reshape(n, h, hq // h, D).permute(1, 0, 2, 3).reshape(h, -1, D)
    mask = seen.repeat_interleave(hq // h, 0)
    s = (torch.bmm(qs, k.transpose(1, 2).contiguous()) * D ** -0.5).masked_fill(~mask, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)  # rows that see nothing
    o, a = torch.bmm(p, v), torch.bmm(p, v.abs())
    size = (torch.bmm(qs.abs(), k.abs().transpose(1, 2).contiguous()) * D ** -0.5).masked_fill(~mask, 0.0)
    e = HALF[dtype] * (a + o.abs()) * (1 + 2.0**-6) + TINY[dtype]
    if dtype == F16:
        e = e + 2.0**-25 * torch.bmm(mask.double().expand(h, -1, -1).contiguous(), v.abs())
    bar = e + U * (320 * size.amax(-1, keepdim=True) + 64 + k.shape[1] / 64) * a
    g = got.double().reshape(n, h, hq // h, D).permute(1, 0, 2, 3).reshape(h, -1, D)
    assert torch.isfinite(g).all(), what
    over = float(((g - o).abs() - bar).max())
    assert over <= 0, (what, over)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("page,hole", [(64, None), (64, 4), (48, 3), (100, 0), (390, 1), (1, 70)])
def test_prefix_of_any_length(gpu, page, hole, dtype):
    """720 rows against prefixes from one key to many tiles a workgroup, whole pages and cut ones, one of
    them not there; what lies behind the prefix's last token is no key, whatever it holds."""
    b, n, hkv, group, longest = 9, 40, 32, 2, 130 if page == 1 else 1700
    n_pre, own = -(-longest // page), 64
    kpool, vpool = (t.to(gpu) for t in _pools(b, hkv, own, dtype, "cpu", 201))
    kpre, vpre = (t.to(gpu) for t in _pools(n_pre, hkv, page, dtype, "cpu", 203))
    ids = torch.randperm(n_pre, generator=_gen(205)).int().to(gpu)
    if hole is not None:
        ids[hole] = -1
    tables, lengths = torch.arange(b, dtype=torch.int32, device=gpu)[:, None].contiguous(), [n + i for i in range(b)]
    q = torch.randn(b, n, hkv * group, D, generator=_gen(206)).to(dtype).to(gpu)
    for prefix in (1, 63, 64, 65, 129, 200, 330, 450, 700, 1100, longest):
        if prefix > longest:
            continue
        print("prefix", page, prefix, dtype, flush=True)
        last, o = int(ids[(prefix - 1) // page]), (prefix - 1) % page + 1
        kp, vp = kpre.clone(), vpre.clone()
        if last >= 0:
            kp[last, 0, :, o:] = float("inf")
            vp[last, 0, :, :, o:] = float("nan")
        got = attend_shared(q, kpool, vpool, tables, _i32(lengths, gpu), page_tokens=own,
                            prefix_pages=ids, prefix_tokens=prefix, prefix_pools=(kp, vp, page))
        k0, v0, there = _listed(kp, vp, page, ids, prefix)
        for i in range(b):
            k1, v1, _ = _listed(kpool, vpool, own, tables[i], lengths[i])
            row = torch.arange(n, device=gpu)[:, None]
            seen = torch.cat((there.expand(n, -1), torch.arange(lengths[i], device=gpu) <= lengths[i] - n + row), 1)
            _check_sequence(got[i], q[i], torch.cat((k0, k1), 1), torch.cat((v0, v1), 1), seen, dtype, (prefix, i))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,padded,prefix", [(64, False, 0), (100, True, 0), (390, False, 70), (48, True, 70)])
def test_many_rows_of_own_keys(gpu, page, padded, prefix, causal):
    """150 rows of 16 sequences against own keys of many tiles a workgroup: tiles that all rows see, then
    those of the causal limit; cut pages, pages that are not there, padding, keys behind the length."""
    b, n, hkv = 16, 150, 16
    width = -(-1100 // page)
    kpool, vpool = (t.to(gpu) for t in _pools(b * width + 2, hkv, page, BF, "cpu", 211))
    tables = torch.randperm(b * width, generator=_gen(213)).int().reshape(b, width).to(gpu)
    ids = _i32([b * width, b * width + 1], gpu)
    lengths = [150 + 61 * i for i in range(b)]  # 150 .. 1065
    new = [n - 9 * i for i in range(b)] if padded else None
    tables[3, 1] = -1
    tables[7, 0] = b * width + 2
    for i, length in enumerate(lengths):
        p, o = int(tables[i, length // page]), length % page
        if 0 <= p < kpool.shape[0]:
            kpool[p, 0, :, o:] = float("inf")
            vpool[p, 0, :, :, o:] = float("nan")
    q = torch.randn(b, n, hkv, D, generator=_gen(214)).to(BF).to(gpu)
    pre = min(prefix, 2 * page)
    got = attend_shared(q, kpool, vpool, tables, _i32(lengths, gpu), page_tokens=page, causal=causal,
                        prefix_pages=ids, prefix_tokens=pre, new_lens=None if new is None else _i32(new, gpu))
    k0, v0, t0 = _listed(kpool, vpool, page, ids, pre)
    for i in range(b):
        m = n if new is None else new[i]
        k1, v1, t1 = _listed(kpool, vpool, page, tables[i], lengths[i])
        row = torch.arange(m, device=gpu)[:, None]
        limit = lengths[i] - m + row if causal else lengths[i] + 0 * row
        seen = torch.cat((t0.expand(m, -1), t1 & (torch.arange(lengths[i], device=gpu) <= limit)), 1)
        _check_sequence(got[i, :m], q[i, :m], torch.cat((k0, k1), 1), torch.cat((v0, v1), 1), seen, BF, i)
        assert not got[i, m:].any()


def test_values_at_the_limit_of_many_rows(gpu):
    """150 rows over 600 own keys: an infinity and a NaN in V of a token reach the rows that see it and no
    earlier ones, behind the tiles that all rows see."""
    b, n, hkv, page = 16, 150, 16, 64
    kpool, vpool = (t.to(gpu) for t in _pools(b * 10, hkv, page, BF, "cpu", 221))
    tables = torch.arange(b * 10, dtype=torch.int32, device=gpu).reshape(b, 10)
    q = torch.randn(b, n, hkv, D, generator=_gen(222)).to(BF).to(gpu)

    def run():
        return attend_shared(q, kpool, vpool, tables, _i32([600] * b, gpu), page_tokens=page)

    clean = run()
    at = 100  # row 100's own token
    p, o = (450 + at) // page, (450 + at) % page
    vpool[tables[:, p].long(), 0, :, 5, o], vpool[tables[:, p].long(), 0, :, 77, o] = float("inf"), float("nan")
    got = run()
    assert torch.equal(got[:, :at], clean[:, :at])
    assert torch.isinf(got[:, at:, :, 5]).all() and torch.isnan(got[:, at:, :, 77]).all()
    rest = [c for c in range(D) if c not in (5, 77)]
    assert torch.equal(got[:, at:][..., rest], clean[:, at:][..., rest])


@pytest.mark.parametrize("prefix,length,new,rows,hq", [(100, 1, None, 1, 4), (129, 130, None, 3, 4), (64, 0, 0, 2, 2),
                                                       (1, 64, 2, 4, 8), (300, 90, None, 1, 2)])
def test_single_sequence_with_few_keys(gpu, prefix, length, new, rows, hq):
    """One sequence whose prefix and own keys one workgroup takes, with a page of each that is not there."""
    page, hkv = 48, 2
    kpool, vpool = _pools(16, hkv, page, BF, "cpu", 231)
    tables, ids = torch.tensor([[3, -1, 5, 6]], dtype=torch.int32), [7, 16, 9, 10, 11, 12, 13]
    q = torch.randn(1, rows, hq, D, generator=_gen(232)).to(BF)
    new = None if new is None else [new]
    want, bar = _attention(q, (kpool, vpool, page, tables), [length], new, True, (kpool, vpool, page, ids, prefix))
    got = attend_shared(q.to(gpu), kpool.to(gpu), vpool.to(gpu), tables.to(gpu), _i32([length], gpu), page_tokens=page,
                        prefix_pages=_i32(ids, gpu), prefix_tokens=prefix, new_lens=None if new is None else _i32(new, gpu))
    _check(got, want, bar)


@pytest.mark.parametrize("b,rows,prefix", [(150, 1, 0), (150, 2, 100), (1100, 2, 64)])
def test_many_short_sequences(gpu, b, rows, prefix):
    """More sequences than CUs (several share a workgroup) and more than the 1024 whose padding rows
    close up, against the same call for one sequence at a time on the first, the last and some between."""
    page, hkv, hq = 16, 2, 4
    kpool, vpool = (t.to(gpu) for t in _pools(2 * b + 7, hkv, page, BF, "cpu", 171))
    tables = torch.randperm(2 * b, generator=_gen(173)).int().reshape(b, 2).to(gpu)
    ids = torch.arange(2 * b, 2 * b + 7, dtype=torch.int32, device=gpu)
    new = [rows if i % 3 else i % 2 for i in range(b)]
    lengths = [min(2 * page, new[i] + (11 * i) % 31) for i in range(b)]
    q = torch.randn(b, rows, hq, D, generator=_gen(174)).to(BF).to(gpu)
    lens, news = _i32(lengths, gpu), _i32(new, gpu)
    got = attend_shared(q, kpool, vpool, tables, lens, page_tokens=page, prefix_pages=ids, prefix_tokens=prefix,
                        new_lens=news)
    for i in [0, 1, 2, b // 2, b // 2 + 1, b - 2, b - 1]:
        want, bar = _attention(q[i:i + 1].cpu(), (kpool.cpu(), vpool.cpu(), page, tables[i:i + 1].cpu()),
                               lengths[i:i + 1], new[i:i + 1], True,
                               (kpool.cpu(), vpool.cpu(), page, ids.tolist(), prefix) if prefix else None)
        _check(got[i:i + 1], want, bar, i)
        assert not got[i, new[i]:].any()


def test_pools_past_32_bit_offsets(gpu):
    """The last pages of pools of more than 2^32 bytes."""
    page, hkv = 64, 8
    n_pages = (1 << 31) // (hkv * page * D) + 40
    kpool = torch.empty(n_pages, 1, hkv, page, D, dtype=BF, device=gpu)
    vpool = torch.empty(n_pages, 1, hkv, D, page, dtype=BF, device=gpu)
    small = [n_pages - 4 + i for i in range(4)]
    k, v = _rows((1, 100, hkv, D), 95, BF, gpu), _rows((1, 100, hkv, D), 96, BF, gpu)
    tables = _i32([small[:2]], gpu)
    append_pages(k, v, kpool, vpool, tables, _i32([100], gpu), page_tokens=page)
    append_pages(k[:, :1], v[:, :1], kpool, vpool, _i32([small[2:]], gpu), _i32([65], gpu), page_tokens=page)
    assert torch.equal(kpool[small[1], 0, :, :36].transpose(0, 1), k[0, 64:])
    assert torch.equal(vpool[small[1], 0, :, :, :36].permute(2, 0, 1), v[0, 64:])
    assert torch.equal(kpool[small[3], 0, :, 0], k[0, 0]) and torch.equal(vpool[small[3], 0, :, :, 0], v[0, 0])
    q = torch.randn(1, 1, hkv, D, generator=_gen(97)).to(BF)
    cpu = (kpool[small].cpu(), vpool[small].cpu())
    want, bar = _attention(q, (*cpu, page, torch.tensor([[0, 1]])), [100], None, True, (*cpu, page, [0, 1], 90))
    got = attend_shared(q.to(gpu), kpool, vpool, tables, _i32([100], gpu), page_tokens=page,
                        prefix_pages=tables[0], prefix_tokens=90)
    _check(got, want, bar)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_rollouts_from_one_history(gpu, dtype):
    """A frame-slot cache of one stream fills, then three rollouts go on from it token by token and in
    a chunk: every step appends (norm and rotation on the way) and attends; against float64 of the
    keys that the caches hold.  The steps run as one captured graph, replayed with lengths that grow
    on the GPU, with eager work between, and equal the eager calls bit for bit."""
    T, hkv, hq, page, chunk_f, b = 40, 2, 4, 16, 2, 3
    cache = make_kv_cache_allocator(num_layers=1, num_heads=hkv, head_dim=D, frame_sequence_length=T,
                                    local_attn_size=5, sink_size=1, num_frame_per_block=chunk_f)(
        1, dtype=BF, device=gpu)[0]
    for c in range(3):
        x = [_rows((1, chunk_f * T, hkv, D), 100 + 3 * c + i, BF, gpu) for i in range(3)]
        _, update = attend_cached(*x, cache, c * chunk_f * T)
        apply_cache_updates([cache], [(0, update)])
    pages, tokens, pools = history_pages(cache)
    assert tokens == 5 * T and pages.tolist() == list(cache.table)
    if dtype != BF:  # the same history in float16 pages
        k, v = cache.logical_kv()
        pools = (*kernels.new_pools(5, 1, hkv, T, dtype, gpu)[:2], T)
        kernels.append_frames(k.to(dtype), v.to(dtype), *pools[:2], list(range(5)), frame_tokens=T)
        pages = torch.arange(5, dtype=torch.int32, device=gpu)
    kpool, vpool, _, _ = kernels.new_pools(b * 4, 1, hkv, page, dtype, gpu)
    tables = torch.randperm(b * 4, generator=_gen(110)).int().reshape(b, 4).to(gpu)
    cos, sin = _tables(tokens + 4 * page, D, gpu)
    wq, wk = _weight(111, torch.float32, gpu), _weight(112, torch.float32, gpu)
    lengths = torch.zeros(b, dtype=torch.int32, device=gpu)

    def step(q, k, v, new=None):
        q = append_pages(k, v, kpool, vpool, tables, lengths, page_tokens=page, new_lens=new, q=q, cos=cos,
                         sin=sin, position0=tokens, norm_q=(wq, EPS), norm_k=(wk, EPS))
        return q, attend_shared(q, kpool, vpool, tables, lengths, page_tokens=page, prefix_pages=pages,
                                prefix_tokens=tokens, prefix_pools=pools, new_lens=new)

    def check(q, got, new):
        want, bar = _attention(q.cpu(), (kpool.cpu(), vpool.cpu(), page, tables.cpu()), lengths.tolist(), new,
                               True, (pools[0].cpu(), pools[1].cpu(), T, pages.tolist(), tokens))
        _check(got, want, bar)

    new = [20, 7, 0]
    lengths += _i32(new, gpu)
    q, got = step(*(_rows((b, 20, h, D), 120 + i, dtype, gpu) for i, h in enumerate((hq, hkv, hkv))),
                  _i32(new, gpu))
    check(q, got, new)
    x = [_rows((b, 1, h, D), 130 + i, dtype, gpu) for i, h in enumerate((hq, hkv, hkv))]

    def token():
        lengths.add_(1)
        return step(*x)

    before = [t.clone() for t in (lengths, kpool, vpool)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token()
    torch.cuda.current_stream().wait_stream(side)
    for t, old in zip((lengths, kpool, vpool), before):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, got = token()
    for i in range(4):
        for j, t in enumerate(x):
            t.copy_(_rows(t.shape, 140 + 3 * i + j, dtype, gpu))
        graph.replay()
        torch.cuda.synchronize()
        check(q, got, None)
        saved = [t.clone() for t in (kpool, vpool, got)]
        eager_q, eager = step(*x)  # the same tokens to the same places
        assert torch.equal(eager, saved[2]) and torch.equal(kpool, saved[0]) and torch.equal(vpool, saved[1])
    assert lengths.tolist() == [24, 11, 4]


def test_two_streams_and_two_graphs(gpu):
    """Calls on two streams side by side, and two graphs of one capturing stream replayed on two."""
    hkv, page, prefix = 4, 64, 3000
    n_pre = -(-prefix // page)
    kpool, vpool = (t.to(gpu) for t in _pools(n_pre + 8, hkv, page, BF, "cpu", 151))
    ids = torch.arange(n_pre, dtype=torch.int32, device=gpu)
    tables = torch.arange(n_pre, n_pre + 8, dtype=torch.int32, device=gpu).reshape(4, 2)
    lengths = _i32([1, 50, 100, 128], gpu)
    qs = [torch.randn(4, 1, 8, D, generator=_gen(152 + i)).to(BF).to(gpu) for i in range(2)]

    def run(q):
        return attend_shared(q, kpool, vpool, tables, lengths, page_tokens=page, prefix_pages=ids,
                             prefix_tokens=prefix)

    want = [run(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(q))
        graphs.append(g)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_no_sequences_and_no_rows(gpu):
    kpool, vpool = _pools(2, 1, 64, BF, gpu, 161)
    before = kpool.clone()
    for shape in ((0, 3, 1, D), (2, 0, 1, D)):
        x = torch.empty(shape, dtype=BF, device=gpu)
        tables, lengths = torch.zeros(shape[0], 1, dtype=torch.int32, device=gpu), _i32([1] * shape[0], gpu)
        assert append_pages(x, x, kpool, vpool, tables, lengths, page_tokens=64, q=x).shape == shape
        assert attend_shared(x, kpool, vpool, tables, lengths, page_tokens=64).shape == shape
    assert torch.equal(kpool.view(torch.int16), before.view(torch.int16))
