"""Per-head q/k RMS norm with the position rotation, and its gradient, against float64.

Bars, per element.  Forward: one rounding to the type (half a step of the value) plus the fp32
arithmetic before it, at most 16 roundings of 2^-24 on each of the pair's two normalised values
(square sum: 7 additions in a lane and 4 across it, mean, rsqrt, two products, two of the
rotation).  dx: the same half step plus at most 32 fp32 roundings on the two terms it subtracts.
dw: at most 256 fp32 roundings on the sum of absolute terms (what a thread, a workgroup and the
last kernel add one after another at these sizes) plus the rounding to the weight's type.
"""

from types import SimpleNamespace

import pytest
import torch

from solarwm_amd import qk_norm_rope

pytestmark = pytest.mark.gpu

D = 128
EPS = 1e-6
U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}  # half a subnormal step
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _tables(rows, rot, dev):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    ang = torch.outer(torch.arange(rows, dtype=torch.float64), inv)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


def _pairs(rot, inter):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)


def _turn(y, cos, sin, rot, inter, back=False):
    """(turned, sum of the absolute values of each channel's pair)."""
    z, size = y.clone(), y.abs()
    if rot:
        i, j = _pairs(rot, inter)
        s = -sin if back else sin
        z[..., i] = y[..., i] * cos - y[..., j] * s
        z[..., j] = y[..., j] * cos + y[..., i] * s
        both = y[..., i].abs() + y[..., j].abs()
        size = size.clone()
        size[..., i] = both
        size[..., j] = both
    return z, size


def _reference(x, w, cos, sin, rot, inter, norm, g=None):
    """float64 on the CPU: z and its size, and with g also dx, its size, dw, its size."""
    x = x.detach().double().cpu()
    w = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    r = 1.0 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) if norm else torch.ones_like(x[..., :1])
    if not norm:
        w = torch.ones_like(w)
    z, zs = _turn(x * r * w, cos, sin, rot, inter)
    if g is None:
        return z, zs
    dy, dys = _turn(g.double().cpu(), cos, sin, rot, inter, back=True)
    u, us = dy * w, dys * w.abs()
    if not norm:
        return z, zs, u, us, None, None
    dx = r * (u - x * r.pow(2) * (u * x).mean(-1, keepdim=True))
    dxs = r * (us + x.abs() * r.pow(2) * (us * x.abs()).mean(-1, keepdim=True))
    terms = dy * x * r
    return z, zs, dx, dxs, terms.flatten(0, -2).sum(0), (dys * x.abs() * r).flatten(0, -2).sum(0)


def _near(what, got, want, size, dtype, roundings):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), what
    bar = HALF[dtype] * want.abs() * (1 + 2.0**-6) + TINY[dtype] + roundings * U * size
    over = (got - want).abs() - bar
    assert float(over.max()) <= 0, (what, float(over.max()), float((got - want).abs().max()))


def _rows(shape, seed, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(*shape[:2], 1, 1, generator=g))
    return x.to(dtype).to(dev)


def _weight(seed, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(dev)


SHAPES = [  # batch, length, q heads, k heads, rotated channels
    (1, 1, 1, 1, 128),
    (1, 1, 40, 8, 96),
    (2, 7, 5, 3, 64),
    (3, 65, 12, 12, 16),
    (1, 300, 6, 2, 112),
    (2, 33, 4, 1, 0),
]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradient(gpu, shape, inter, dtype):
    b, n, hq, hk, rot = shape
    print("qk_norm_rope", shape, inter, dtype, flush=True)
    q, k = _rows((b, n, hq, D), 1, dtype, gpu), _rows((b, n, hk, D), 2, dtype, gpu)
    wq, wk = _weight(3, F32, gpu), _weight(4, dtype, gpu)
    gq, gk = _rows((b, n, hq, D), 5, dtype, gpu), _rows((b, n, hk, D), 6, dtype, gpu)
    cos, sin = _tables(n + 5, rot, gpu) if rot else (None, None)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    zq, zk = qk_norm_rope(q, k, cos, sin, norm_q=SimpleNamespace(weight=wq, eps=EPS), norm_k=(wk, EPS),
                          position0=5 if rot else 0, interleaved=inter)
    dq, dk, dwq, dwk = torch.autograd.grad((zq, zk), leaves, (gq, gk))
    c, s = (t[5:, None].double().cpu() for t in (cos, sin)) if rot else (None, None)
    for name, x, w, g, z, dx, dw in (("q", q, wq, gq, zq, dq, dwq), ("k", k, wk, gk, zk, dk, dwk)):
        z_, zs, dx_, dxs, dw_, dws = _reference(x, w, c, s, rot, inter, True, g)
        _near(name, z, z_, zs, dtype, 16)
        _near("d" + name, dx, dx_, dxs, dtype, 32)
        assert dw.dtype == w.dtype
        _near("dw" + name, dw, dw_, dws, w.dtype, 256)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("norm_q,norm_k", [(True, False), (False, True), (False, False)])
def test_norm_of_one_side(gpu, norm_q, norm_k, dtype):
    q, k = _rows((2, 9, 3, D), 11, dtype, gpu), _rows((2, 9, 2, D), 12, dtype, gpu)
    gq, gk = _rows((2, 9, 3, D), 13, dtype, gpu), _rows((2, 9, 2, D), 14, dtype, gpu)
    cos, sin = _tables(9, 64, gpu)
    q.requires_grad_(), k.requires_grad_()
    zq, zk = qk_norm_rope(q, k, cos, sin, norm_q=(None, EPS) if norm_q else None,
                          norm_k=(None, EPS) if norm_k else None)
    dq, dk = torch.autograd.grad((zq, zk), (q, k), (gq, gk))
    c, s = cos[:, None].double().cpu(), sin[:, None].double().cpu()
    for x, g, z, dx, norm in ((q, gq, zq, dq, norm_q), (k, gk, zk, dk, norm_k)):
        z_, zs, dx_, dxs, _, _ = _reference(x, None, c, s, 64, False, norm, g)
        _near("z", z, z_, zs, dtype, 16)
        _near("dx", dx, dx_, dxs, dtype, 32)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_slices_of_one_projection(gpu, dtype):
    """q and k as slices of a packed projection, tables as slices of wider ones, gradients that are
    expanded or transposed: the same bits as contiguous tensors give."""
    x = _rows((2, 37, 4 + 2 * 2, D), 21, dtype, gpu)
    q, k = x[:, :, :4].detach().requires_grad_(), x[:, :, 4:6].detach().requires_grad_()
    wide = torch.cat(_tables(37, 96, gpu), 1)
    cos, sin = wide[:, :48], wide[:, 48:]
    w = _weight(22, F32, gpu).requires_grad_()
    gq = _rows((37, 2, 4, D), 23, dtype, gpu).transpose(0, 1)
    gk = _rows((2, 37, 1, D), 24, dtype, gpu).expand(2, 37, 2, D)

    def run(q, k, cos, sin, gq, gk):
        z = qk_norm_rope(q, k, cos, sin, norm_q=(w, EPS), norm_k=(w, EPS))
        return (*z, *torch.autograd.grad(z, (q, k, w), (gq, gk)))

    got = run(q, k, cos, sin, gq, gk)
    want = run(q.detach().clone(memory_format=torch.contiguous_format).requires_grad_(),
               k.detach().clone(memory_format=torch.contiguous_format).requires_grad_(),
               cos.contiguous(), sin.contiguous(), gq.contiguous(), gk.contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions(gpu, kind, inter):
    """Positions per token, shared or per sequence; rows outside the table turn to NaN in their
    rotated channels and nowhere else, and infinities behind the rotated channels stay there."""
    b, n, rot = 3, 21, 64
    q = _rows((b, n, 2, D), 31, F32, gpu)
    cos, sin = _tables(50, rot, gpu)
    pos = torch.randint(0, 45, (b, n), generator=torch.Generator().manual_seed(32)).to(kind)
    pos[1, 4], pos[2, 0] = 46, -6
    z, none = qk_norm_rope(q, None, cos, sin, norm_q=(None, EPS), positions=pos.to(gpu), position0=5,
                           interleaved=inter)
    assert none is None
    at = pos.long() + 5
    bad = (at < 0) | (at >= 50)
    assert int(bad.sum()) == 2
    assert torch.isnan(z[bad.to(gpu)][..., :rot]).all()
    assert torch.isfinite(z[bad.to(gpu)][..., rot:]).all()
    c, s = (t.cpu().double()[at.clamp(0, 49)][:, :, None] for t in (cos, sin))
    z_, zs = _reference(q, None, c, s, rot, inter, True)
    ok = ~bad
    _near("z", z.cpu()[ok], z_[ok], zs[ok], F32, 16)
    shared, _ = qk_norm_rope(q, None, cos, sin, norm_q=(None, EPS), positions=pos[0].to(gpu), position0=5,
                             interleaved=inter)
    per_row, _ = qk_norm_rope(q, None, cos, sin, norm_q=(None, EPS), positions=pos[:1].expand(b, n).to(gpu),
                              position0=5, interleaved=inter)
    assert torch.equal(shared, per_row)
    q[0, 0, 0, rot + 3] = float("inf")
    q[0, 1, 0, 2] = float("nan")
    z, _ = qk_norm_rope(q, None, cos, sin, interleaved=inter)
    assert z[0, 0, 0, rot + 3] == float("inf") and torch.isfinite(z[0, 0, 0, :rot]).all()
    assert int(torch.isnan(z[0, 1, 0]).sum()) == 2 and torch.isfinite(z[0, 2:]).all()


def test_zero_rows_and_no_tokens(gpu):
    q = torch.zeros(1, 3, 2, D, device=gpu, dtype=BF).requires_grad_()
    w = _weight(41, F32, gpu).requires_grad_()
    cos, sin = _tables(3, 128, gpu)
    z, _ = qk_norm_rope(q, None, cos, sin, norm_q=(w, EPS))
    dq, dw = torch.autograd.grad(z, (q, w), torch.ones_like(z))
    assert torch.equal(z, torch.zeros_like(z)) and torch.equal(dw, torch.zeros_like(dw))
    assert torch.isfinite(dq).all()
    for shape in ((0, 3, 2, D), (2, 0, 2, D)):
        e = torch.empty(shape, device=gpu, dtype=BF).requires_grad_()
        z, zk = qk_norm_rope(e, e, cos, sin, norm_q=(w, EPS), norm_k=(w, EPS))
        de, dw = torch.autograd.grad((z, zk), (e, w), (torch.empty_like(z), torch.empty_like(zk)))
        assert z.shape == zk.shape == de.shape == e.shape
        assert torch.equal(dw, torch.zeros_like(dw))


def test_gradient_against_differences(gpu):
    """dL along random directions of q, k and the weights: the kernel's gradient against central
    differences of the float64 definition.  The difference's own error is h^2 f''' ~ 1e-7 of the
    terms; float32 gradients add 32 (dx) and 256 (dw) roundings of 2^-24 on the absolute terms,
    2e-5 of them at most; the bar is 1e-4 of the sum of absolute terms."""
    b, n, hq, hk, rot = 2, 5, 3, 2, 96
    q, k = _rows((b, n, hq, D), 51, F32, gpu), _rows((b, n, hk, D), 52, F32, gpu)
    wq, wk = _weight(53, F32, gpu), _weight(54, F32, gpu)
    gq, gk = _rows((b, n, hq, D), 55, F32, gpu), _rows((b, n, hk, D), 56, F32, gpu)
    cos, sin = _tables(n, rot, gpu)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    z = qk_norm_rope(q, k, cos, sin, norm_q=(wq, EPS), norm_k=(wk, EPS))
    grads = [t.double().cpu() for t in torch.autograd.grad(z, leaves, (gq, gk))]
    at = [t.detach().double().cpu() for t in leaves]
    c, s = cos[:, None].double().cpu(), sin[:, None].double().cpu()

    def loss(q, k, wq, wk):
        zq, _ = _reference(q, wq, c, s, rot, False, True)
        zk, _ = _reference(k, wk, c, s, rot, False, True)
        return (zq * gq.double().cpu()).sum() + (zk * gk.double().cpu()).sum()

    h = 1e-5
    for i in range(4):
        d = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(60 + i), dtype=torch.float64)
        up, down = ([x + sign * h * d if j == i else x for j, x in enumerate(at)] for sign in (1, -1))
        want = float((loss(*up) - loss(*down)) / (2 * h))
        got, size = float((grads[i] * d).sum()), float((grads[i] * d).abs().sum())
        assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_same_bits_every_time_and_on_another_stream(gpu):
    q = _rows((2, 4000, 6, D), 71, BF, gpu).requires_grad_()
    k = _rows((2, 4000, 2, D), 72, BF, gpu).requires_grad_()
    w = _weight(73, F32, gpu).requires_grad_()
    cos, sin = _tables(4000, 128, gpu)

    def run():
        z = qk_norm_rope(q, k, cos, sin, norm_q=(w, EPS), norm_k=(w, EPS), interleaved=True)
        return (*z, *torch.autograd.grad(z, (q, k, w), z))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_long_weight_gradient(gpu):
    """Enough rows for every workgroup to loop: dw against float64, 4 * 4000 * 12 / (16 * 2048)
    rounds of 4 heads per thread stay below the 256 roundings of the bar."""
    q = _rows((4, 4000, 48, D), 81, BF, gpu).requires_grad_()
    w = _weight(82, F32, gpu).requires_grad_()
    cos, sin = _tables(4000, 128, gpu)
    g = _rows((4, 4000, 48, D), 83, BF, gpu)
    z, _ = qk_norm_rope(q, None, cos, sin, norm_q=(w, EPS))
    dw, = torch.autograd.grad(z, w, g)
    x, gd = q.detach().double(), g.double()
    c, s = cos[:, None].double(), sin[:, None].double()
    i, j = (t.to(gpu) for t in _pairs(128, False))
    dy = gd.clone()
    dy[..., i] = gd[..., i] * c + gd[..., j] * s
    dy[..., j] = gd[..., j] * c - gd[..., i] * s
    terms = dy * x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    want, size = terms.flatten(0, -2).sum(0).cpu(), terms.abs().flatten(0, -2).sum(0).cpu()
    # |dy| is bounded by the pair's two terms, so its size is at most sqrt(2) of |dy| on average
    _near("dw", dw, want, 2 * size, F32, 256)


def test_graph_replays(gpu):
    """Forward and backward captured once and replayed on new inputs, with eager work between."""
    q = _rows((1, 50, 4, D), 91, BF, gpu).requires_grad_()
    k = _rows((1, 50, 2, D), 92, BF, gpu).requires_grad_()
    w = _weight(93, F32, gpu).requires_grad_()
    g = _rows((1, 50, 4, D), 94, BF, gpu)
    gk = _rows((1, 50, 2, D), 95, BF, gpu)
    cos, sin = _tables(50, 128, gpu)

    def run():
        z = qk_norm_rope(q, k, cos, sin, norm_q=(w, EPS), norm_k=(w, EPS))
        return (*(t.detach() for t in z), *torch.autograd.grad(z, (q, k, w), (g, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        with torch.no_grad():
            q.copy_(_rows((1, 50, 4, D), 100 + i, BF, gpu))
            g.copy_(_rows((1, 50, 4, D), 200 + i, BF, gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
