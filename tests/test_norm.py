"""The root-mean-square norm, its residual and 8-bit output, and its gradient against
64-bit arithmetic.

u = 2^-24. A row's sum of squares has at most 32 terms a thread and 10 levels of a tree
over the threads, all positive, and h is off by u of itself, so the sum is off by
(32 + 10 + 2) u of itself; the mean, eps and the root leave r off by 25 u at most, and y
has two products and h's own rounding more: |y - exact| <= 29 u |y| < 2^-19 |y|, and the
output's type adds half a step of it. A scale follows y's largest magnitude, with one
rounding more. A code is off by half a step of its value (2^-4 in e4m3, 2^-3 in e5m2) or,
below the normal range, by half the smallest step times the scale.

The gradient: with a = w dy and M = r^2 mean |a h|, the mean of a h is off by 44 u M / r^2,
the product k = r^2 mean(a h) by (44 + 2 * 25 + 4) u M, and dx = r (a - h k) + dres by less
than 128 u r (|a| + |h| M) + 2 u (|dx| + |dres|) besides its type's rounding. A term of
dw is off by 28 u, and the R additions that an element takes at most by R u of the terms'
magnitudes.
"""
import numpy as np
import pytest
import torch

import mantle_cuda as M
from fp8_reference import CODE, TOP, up16

u = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F, H = torch.float32, torch.bfloat16
ptr = lambda n, at=1 << 20: M.DevicePtr(at, n)  # noqa: E731
BIG = ptr(1 << 40)


# ── refusals (no launch) ─────────────────────────────────────────────────────
def n_args(r, c, kind=0, wkind=0, fmt=0, pow2=0, eps=1e-6, **change):
    per, perw = (2 if k == 1 else 4 for k in (kind, wkind))
    a = dict(y=ptr(r * c * per), q=None, s=None, h=None, x=ptr(r * c * per), res=None, w=ptr(c * perw))
    a.update(change)
    return [*a.values(), c, kind, wkind, fmt, pow2, eps]


@pytest.mark.parametrize("args,nd,match", [
    (n_args(4, 100, y=None), 4, "give y, the codes"),
    (n_args(4, 100, q=BIG), 4, "go together"),
    (n_args(4, 100, s=BIG), 4, "go together"),
    (n_args(4, 100, h=BIG), 4, "without a residual"),
    (n_args(4, 100), 5, "y: 1600 bytes, the launch touches 2000"),
    (n_args(4, 100, x=ptr(1599)), 4, "the input"),
    (n_args(4, 100, w=ptr(399)), 4, "the weights"),
    (n_args(4, 100, wkind=1, w=ptr(199)), 4, "the weights"),
    (n_args(4, 100, res=ptr(1599)), 4, "the residual"),
    (n_args(4, 100, res=BIG, h=ptr(1599)), 4, "h: "),
    (n_args(4, 100, q=ptr(4 * 112 - 1), s=BIG), 4, "the codes"),
    (n_args(4, 129, q=BIG, s=ptr(31)), 4, "the scales"),
    (n_args(4, 100, q=ptr(1 << 20, (1 << 20) + 8), s=BIG), 4, "the codes must be 16-byte"),
    (n_args(4, 100, x=ptr(1 << 20, (1 << 20) + 2)), 4, "the input must be 4-byte"),
    (n_args(4, 100, kind=2), 4, "must be 0 or 1"),
    (n_args(4, 100, wkind=-1), 4, "must be 0 or 1"),
    (n_args(4, 100, fmt=2), 4, "must be 0 or 1"),
    (n_args(4, 100, pow2=3), 4, "must be 0 or 1"),
    (n_args(4, 100, eps=-1e-6), 4, "eps"),
    (n_args(4, 100, eps=float("nan")), 4, "eps"),
    (n_args(4, 100, eps=float("inf")), 4, "eps"),
    (n_args(4, -1), 4, "negative"),
    (n_args(4, 32769, y=BIG, x=BIG, w=BIG), 4, "more than 32768 columns"),
    (n_args(4, 100, x=ptr(0, 0)), 4, "the input must be a device buffer"),
    (n_args(4, 100, w=ptr(0, 0)), 4, "the weights must be a device buffer"),
    (n_args(4, 100, res=ptr(0, 0)), 4, "the residual must be a device buffer"),
    (n_args(4, 100), (4, 2), "one-dimensional"),
    (n_args(4, 100, eps=1e300), 4, "no Float32"),
    (n_args(4, 100)[:-1], 4, "takes 13 arguments"),
])
def test_rms_norm_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.rms_norm, args, nd)


def g_args(r, c, kind=0, wkind=0, eps=1e-6, **change):
    per, perw = (2 if k == 1 else 4 for k in (kind, wkind))
    a = dict(dx=ptr(r * c * per), dw=None, dy=ptr(r * c * per), h=ptr(r * c * per), w=ptr(c * perw), dres=None)
    a.update(change)
    return [*a.values(), c, kind, wkind, eps]


@pytest.mark.parametrize("args,nd,match", [
    (g_args(4, 100), 5, "dx: 1600 bytes"),
    (g_args(4, 100, dy=ptr(1599)), 4, "dy"),
    (g_args(4, 100, h=ptr(1599)), 4, "h: "),
    (g_args(4, 100, w=ptr(399)), 4, "the weights"),
    (g_args(4, 100, dres=ptr(1599)), 4, "the residual path"),
    (g_args(4, 100, dw=ptr(399)), 4, "dw: 399"),
    (g_args(4, 100, dw=ptr(400)), 4, "of scratch"),
    (g_args(4, 100, kind=2), 4, "must be 0 or 1"),
    (g_args(4, 100, wkind=2), 4, "must be 0 or 1"),
    (g_args(4, 100, eps=-1.0), 4, "eps"),
    (g_args(4, 40000, dx=BIG, dy=BIG, h=BIG, w=BIG), 4, "more than 32768"),
    (g_args(4, 100, dx=ptr(0, 0)), 4, "dx must be a device buffer"),
])
def test_rms_norm_grad_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.rms_norm_grad, args, nd)


def test_the_gradients_scratch_is_asked_for():
    need = M.workspace_bytes(M.kernels.rms_norm_grad, g_args(4000, 100, dw=ptr(400)), 4000)
    assert need and need % 400 == 0
    assert M.workspace_bytes(M.kernels.rms_norm_grad, g_args(4000, 100), 4000) == 0
    assert M.workspace_bytes(M.kernels.rms_norm_grad, g_args(0, 100, dw=ptr(400)), 0) == 0
    for scratch in (ptr(need - 1), ptr(need, (1 << 20) + 4)):
        with pytest.raises(M.ArgumentError, match="of scratch"):
            M.launch(M.kernels.rms_norm_grad, g_args(4000, 100, dw=ptr(400)), 4000, workspace=scratch)
    with pytest.raises(M.ArgumentError, match="cannot pass"):
        M.launch(M.kernels.rms_norm_grad, g_args(4000, 100, dw=ptr(400)), 4000, workspace=[1, 2])


# ── on the device ────────────────────────────────────────────────────────────
def stream():
    return torch.cuda.current_stream().cuda_stream


def rows(r, c, kind, seed, at=0):
    """A contiguous (r, c) tensor whose first value is `at` values behind an aligned address."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.randn(r * c + at, generator=g).to(kind).cuda()
    return flat[at:].view(r, c)


def norm(x, w, res=None, y=True, h=None, fmt=None, pow2=0, eps=1e-6, out=None):
    r, c = x.shape
    y = (torch.full_like(x, float("nan")) if out is None else out) if y else None
    h = torch.full_like(x, float("nan")) if res is not None and h is None else h
    q = torch.full((r, up16(c)), 255, dtype=torch.uint8, device="cuda") if fmt is not None else None
    s = torch.full((-(-c // 128), r), float("nan"), device="cuda") if fmt is not None else None
    M.launch(M.kernels.rms_norm, (y, q, s, h, x, res, w, c, int(x.dtype == H), int(w.dtype == H), fmt or 0, pow2, eps), r, stream=stream())
    torch.cuda.synchronize()
    return y, h, None if q is None else q.view(CODE[fmt]), s


def exact(x, w, res=None, eps=1e-6):
    h = x.double().cpu() if res is None else x.double().cpu() + res.double().cpu()
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double().cpu()


def check_y(got, want, tol=2.0 ** -19):
    assert ((got.double().cpu() - want).abs() <= (tol + HALF[got.dtype] * (1 + tol)) * want.abs() + 1e-40).all()


def check_codes(q, s, want, fmt, pow2):
    r, c = want.shape
    tol, blocks = 2.0 ** -18, -(-c // 128)
    a = torch.stack([want[:, 128 * b:128 * b + 128].abs().amax(1) for b in range(blocks)]).clamp(min=2.0 ** -96)
    s = s.double().cpu()
    if pow2:
        assert (torch.frexp(s)[0] == 0.5).all() and (a <= TOP[fmt] * s * (1 + tol)).all() and (a > TOP[fmt] / 2 * s * (1 - tol)).all()
    else:
        assert ((s - a / TOP[fmt]).abs() <= tol * a / TOP[fmt]).all()
    each = s.t().repeat_interleave(128, 1)[:, :c]
    v = q.double().cpu()
    half, low = ((2.0 ** -4, 2.0 ** -10), (2.0 ** -3, 2.0 ** -17))[fmt]
    assert ((v[:, :c] * each - want).abs() <= torch.maximum(half * want.abs(), low * each) * (1 + tol) + tol * want.abs()).all()
    assert (q.view(torch.uint8)[:, c:] == 0).all()


SIZES = [(1, 1), (1, 8), (3, 64), (5, 127), (7, 128), (2, 129), (9, 256), (6, 264), (4, 512), (3, 1000), (5, 1024), (3, 1032), (4, 2048),
         (3, 2056), (2, 4013), (3, 4096), (2, 4104), (2, 8192), (1, 8200), (2, 16384), (1, 16392), (2, 20001), (1, 32768), (700, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,wkind", [(F, F), (H, H), (H, F), (F, H)])
@pytest.mark.parametrize("r,c", SIZES)
def test_norm(dev, r, c, kind, wkind):
    w = (1 + 0.3 * rows(1, c, F, 5)[0]).to(wkind)
    for at in (0, 1):  # rows that start on 16 bytes, and rows that do not
        x, res = 3 * rows(r, c, kind, 1, at), rows(r, c, kind, 2, at)
        y, _, _, _ = norm(x, w)
        check_y(y, exact(x, w)[1])
        y, h, _, _ = norm(x, w, res)
        want = exact(x, w, res)
        check_y(h, want[0], 0)
        check_y(y, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("r,c", [(5, 1), (9, 127), (17, 264), (3, 1000), (4, 1024), (9, 2047), (17, 4096), (2, 8192), (3, 8193), (1, 32767), (2, 32768)])
def test_tensors_that_all_start_off_16_bytes(dev, r, c, kind):
    # every tensor as far behind 16 bytes as the others, the outputs among them, and nothing written around them
    w = (1 + 0.3 * rows(1, c, F, 5)[0]).to(kind)
    for at in (1, 3):
        x, res, dy = (rows(r, c, kind, k, at) for k in (1, 2, 3))
        flat = [torch.full((r * c + at + 9,), 7.0, dtype=kind, device="cuda") for _ in range(3)]
        y, h, dx = (f[at:at + r * c].view(r, c) for f in flat)
        _, _, q, s = norm(x, w, res, out=y, h=h, fmt=0)
        want = exact(x, w, res)
        check_y(h, want[0], 0)
        check_y(y, want[1])
        check_codes(q, s, want[1], 0, 0)
        dw = grad(dy, h, w, res, dx=dx)[1]
        dx2, dw2 = grad(*(v.clone() for v in (dy, h, w, res)))
        # cut elsewhere, so summed in another order: each within the bounds of test_norm_grad of the exact value
        a = dy.double() * w.double()
        rr = 1 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + 1e-6)
        m = rr * rr * (a * h.double()).abs().mean(1, keepdim=True)
        tol = 256 * u * rr * (a.abs() + h.double().abs() * m) + 4 * u * (dx2.double().abs() + res.double().abs())
        assert ((dx.double() - dx2.double()).abs() <= tol + 2 * HALF[kind] * dx2.double().abs()).all()
        assert ((dw.double() - dw2.double()).abs() <= 2 * (28 + r) * u * (dy.double() * h.double() * rr).abs().sum(0)).all()
        for f in flat:
            assert (f[:at] == 7).all() and (f[at + r * c:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pow2", [0, 1])
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("r,c", SIZES)
def test_norm_in_8_bits(dev, r, c, kind, fmt, pow2):
    w = (1 + 0.3 * rows(1, c, F, 5)[0]).to(kind)
    for at in (0, 1):
        x, res = rows(r, c, kind, 1, at) * (1 + 30 * (rows(1, c, F, 3) > 2)).to(kind), rows(r, c, kind, 2, at)
        y, h, q, s = norm(x, w, res, fmt=fmt, pow2=pow2)
        want = exact(x, w, res)
        check_y(y, want[1])
        check_codes(q, s, want[1], fmt, pow2)
        only = norm(x, w, res, y=False, fmt=fmt, pow2=pow2)  # the same codes with fewer outputs
        assert torch.equal(only[2].view(torch.uint8), q.view(torch.uint8)) and torch.equal(only[3], s) and torch.equal(only[1], h)


@pytest.mark.gpu
def test_codes_are_the_quantizers_of_y_in_32_bits(dev):
    # the fused codes and scales are what quantize_fp8 makes of the 32-bit y, to the bit
    for r, c in ((37, 1160), (37, 1161), (5, 200), (6, 333)):
        x, w = rows(r, c, F, 1), rows(1, c, F, 2)[0]
        for fmt, pow2 in ((0, 0), (0, 1), (1, 0), (1, 1)):
            y, _, q, s = norm(x, w, fmt=fmt, pow2=pow2)
            q2, s2 = torch.empty_like(q.view(torch.uint8)), torch.empty_like(s)
            M.launch(M.kernels.quantize_fp8, (q2, s2, None, None, y, None, r, c, r, 1, 0, fmt, pow2), 1, stream=stream())
            torch.cuda.synchronize()
            assert torch.equal(q2, q.view(torch.uint8)) and torch.equal(s2, s)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("c", [96, 1000, 4096, 4097])
def test_rows_that_are_not_numbers_stay_apart(dev, kind, c):
    x, w = rows(6, c, kind, 1), torch.ones(c, device="cuda")
    clean = norm(x, w, fmt=0)
    x[1, 3], x[3, c - 1] = float("nan"), float("inf")
    x[4] = 0
    y, _, q, s = norm(x, w, fmt=0)
    y, q, s = y.float(), q.float(), s.t()
    for r in (0, 2, 5):
        assert torch.equal(y[r], clean[0][r].float()) and torch.equal(q[r], clean[2].float()[r]) and torch.equal(s[r], clean[3].t()[r])
    assert y[1].isnan().all() and q[1, :c].isnan().all() and s[1].isnan().all()
    assert y[3, c - 1].isnan() and s[3, -1].isnan()  # infinity / infinity; finite values are zeros
    assert (y[3, :c - 1] == 0).all()
    assert (y[4] == 0).all() and (q[4] == 0).all()  # eps keeps a row of zeros zeros
    assert (q[:, c:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("c", [1, 200, 4096, 4099, 32768])
def test_squares_that_pass_32_bits_together(dev, kind, c):
    # a row on each side of the limit of its sum of squares, 3.4e38, between two others
    top = (2 - 2.0 ** -23) * 2.0 ** 127
    sign = torch.sign(rows(1, c, F, 1)[0] + 1e-3)
    x, w = rows(4, c, kind, 2), (1 + 0.3 * rows(1, c, F, 5)[0])
    x[1], x[2] = (sign * (0.8 * top / c) ** 0.5).to(kind), (sign * (1.25 * top / c) ** 0.5).to(kind)
    square = (x.double() ** 2).sum(1)
    assert square[1] < 0.9 * top and square[2] > 1.1 * top
    y, _, q, s = norm(x, w, fmt=0)
    want = exact(x, w)[1]
    rest = [0, 1, 3]
    check_y(y[rest], want[rest])
    check_codes(q[rest], s[:, rest].contiguous(), want[rest], 0, 0)
    assert (y[2] == 0).all() and (q[2].float() == 0).all()
    dy, dres = rows(4, c, kind, 3), rows(4, c, kind, 4)
    dx, dw = grad(dy, x, w, dres)
    assert torch.equal(dx[2], dres[2])
    only = dy.clone()
    only[2] = 0  # the row gives dw nothing
    check_grad(dx[rest], dw, dy[rest], x[rest], w, dres[rest])
    assert torch.equal(grad(only, x, w, dres)[1], dw)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [64, 4099])
def test_eps_0(dev, c):
    x, w = rows(4, c, F, 2), torch.ones(c, device="cuda")
    x[1], x[2] = 0, 1e-25
    y = norm(x, w, eps=0.0)[0]
    check_y(y[[0, 3]], exact(x, w, eps=0.0)[1][[0, 3]])
    assert y[1].isnan().all() and (y[2] == float("inf")).all()


@pytest.mark.gpu
def test_norm_in_place(dev):
    # h over the residual or over x, y over x
    for c in (200, 4096, 5000):
        for kind in (F, H):
            x, res, w = rows(9, c, kind, 1), rows(9, c, kind, 2), rows(1, c, F, 3)[0]
            y, h, _, _ = norm(x, w, res)
            for over in ("res", "x"):
                x1, r1 = x.clone(), res.clone()
                y2, h2, _, _ = norm(x1, w, r1, h=r1 if over == "res" else x1)
                assert torch.equal(y2, y) and torch.equal(h2, h) and torch.equal(r1 if over == "res" else x1, h)
            x1 = x.clone()
            assert torch.equal(norm(x1, w, res, out=x1)[1], h) and torch.equal(x1, y)


def grad(dy, h, w, dres=None, dw=True, eps=1e-6, dx=None):
    r, c = h.shape
    dx = torch.full_like(h, float("nan")) if dx is None else dx
    dw = torch.full((c,), float("nan"), device="cuda") if dw else None
    args = (dx, dw, dy, h, w, dres, c, int(h.dtype == H), int(w.dtype == H), eps)
    need = M.workspace_bytes(M.kernels.rms_norm_grad, args, r)
    scratch = torch.full((need // 4,), float("nan"), device="cuda") if need else None
    M.launch(M.kernels.rms_norm_grad, args, r, stream=stream(), workspace=scratch)
    torch.cuda.synchronize()
    return dx, dw


@pytest.mark.gpu
@pytest.mark.parametrize("kind,wkind", [(F, F), (H, H), (H, F), (F, H)])
@pytest.mark.parametrize("r,c", SIZES + [(1500, 264), (900, 2056)])
def test_norm_grad(dev, r, c, kind, wkind):
    w = (1 + 0.3 * rows(1, c, F, 5)[0]).to(wkind)
    for at in (0, 1):
        h, dy, dres = 2 * rows(r, c, kind, 1, at), rows(r, c, kind, 2, at), rows(r, c, kind, 3, at)
        for add in (None, dres):
            dx, dw = grad(dy, h, w, add)
            H64, G, W64 = h.double().cpu(), dy.double().cpu(), w.double().cpu()
            rr = 1 / torch.sqrt((H64 * H64).mean(1, keepdim=True) + 1e-6)
            a = G * W64
            want = rr * (a - H64 * rr * rr * (a * H64).mean(1, keepdim=True))
            m = rr * rr * (a * H64).abs().mean(1, keepdim=True)
            d = 0 if add is None else add.double().cpu()
            tol = 128 * u * rr * (a.abs() + H64.abs() * m) + 2 * u * ((want + d).abs() + (0 if add is None else d.abs()))
            tol = tol + HALF[kind] * ((want + d).abs() + tol)
            assert ((dx.double().cpu() - want - d).abs() <= tol).all()
            n = G * H64 * rr
            assert ((dw.double().cpu() - n.sum(0)).abs() <= (28 + r) * u * n.abs().sum(0)).all()
        alone, none = grad(dy, h, w, dres, dw=False)
        assert none is None and torch.equal(alone, dx)


def check_grad(dx, dw, dy, h, w, dres):
    """The bounds at the top, in 64 bits on the device."""
    H64, G, W64 = h.double(), dy.double(), w.double()
    rr = 1 / torch.sqrt((H64 * H64).mean(1, keepdim=True) + 1e-6)
    a = G * W64
    want = rr * (a - H64 * rr * rr * (a * H64).mean(1, keepdim=True))
    m = rr * rr * (a * H64).abs().mean(1, keepdim=True)
    d = torch.zeros_like(want) if dres is None else dres.double()
    tol = 128 * u * rr * (a.abs() + H64.abs() * m) + 2 * u * ((want + d).abs() + d.abs())
    assert ((dx.double() - want - d).abs() <= tol + HALF[h.dtype] * ((want + d).abs() + tol)).all()
    n = G * H64 * rr
    assert ((dw.double() - n.sum(0)).abs() <= (28 + len(h)) * u * n.abs().sum(0)).all()


# more rows than the CTAs take at once, at every count of threads a row, on 16 bytes and cut
TURNS = [(5000, 200), (5000, 201), (3100, 500), (3100, 333), (2000, 1000), (2000, 777), (2000, 1001), (1300, 1504), (1300, 1501), (700, 3001), (700, 4099),
         (1023, 5001), (400, 6001), (400, 7168), (300, 9001), (300, 12001), (300, 16384), (300, 20001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,wkind", [(F, F), (H, H), (H, F)])
@pytest.mark.parametrize("r,c", TURNS)
def test_norm_grad_over_several_turns(dev, r, c, kind, wkind):
    # a CTA's second and later rows: the ring filled again, rows a multiple of eight apart cut alike
    w = (1 + 0.3 * rows(1, c, F, 5)[0]).to(wkind)
    h, dy, dres = 2 * rows(r, c, kind, 1), rows(r, c, kind, 2), rows(r, c, kind, 3)
    for add in (None, dres):
        ctas = M.workspace_bytes(M.kernels.rms_norm_grad, (h, w.float(), dy, h, w, add, c, int(kind == H), int(wkind == H), 1e-6), r) // (4 * c)
        assert 0 < ctas * (4 if c <= 1024 else 1) < r
        dx, dw = grad(dy, h, w, add)
        check_grad(dx, dw, dy, h, w, add)
        again = grad(dy, h, w, add)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
        alone, none = grad(dy, h, w, add, dw=False)
        assert none is None and torch.equal(alone, dx)
        ins = [dy.clone(), h.clone()] + ([] if add is None else [add.clone()])
        for over in range(len(ins)):  # dx over an input
            new = [t.clone() for t in ins]
            got = grad(new[0], new[1], w, new[2] if add is not None else None, dx=new[over])
            assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    for at in (1, 3):  # every tensor as far behind 16 bytes, and only dx
        shift = lambda t: torch.cat([torch.zeros(at, dtype=kind, device="cuda"), t.reshape(-1)])[at:].view(r, c)  # noqa: E731
        flat = torch.full((r * c + at + 9,), 7.0, dtype=kind, device="cuda")
        out = flat[at:at + r * c].view(r, c)
        for ins in ((shift(dy), shift(h), shift(dres)), (dy, h, dres)):
            got = grad(*ins[:2], w, ins[2], dx=out)
            check_grad(got[0], got[1], dy, h, w, dres)
            assert (flat[:at] == 7).all() and (flat[at + r * c:] == 7).all()


@pytest.mark.gpu
def test_norm_grad_against_differences(dev):
    # 64-bit central differences of sum(dy y) with a step of 1e-5: off by 1e-10 of third derivatives, and 1e-11 of rounding
    r, c, e = 3, 24, 1e-5
    h, dy, w = (rows(*s, F, k).double().cpu() for k, s in enumerate(((r, c), (r, c), (1, c))))
    w = w[0]
    loss = lambda hh, ww: (dy * hh / torch.sqrt((hh * hh).mean(1, keepdim=True) + 1e-6) * ww).sum()  # noqa: E731
    dx, dw = grad(dy.float().cuda(), h.float().cuda(), w.float().cuda())
    for i in range(r):
        for j in range(c):
            step = torch.zeros_like(h)
            step[i, j] = e
            assert abs((loss(h + step, w) - loss(h - step, w)).item() / (2 * e) - dx[i, j].item()) < 1e-5
    for j in range(c):
        step = torch.zeros_like(w)
        step[j] = e
        assert abs((loss(h, w + step) - loss(h, w - step)).item() / (2 * e) - dw[j].item()) < 1e-5


@pytest.mark.gpu
def test_norm_grad_in_place_and_repeated(dev):
    for r, c in ((50, 300), (500, 4096), (41, 4099)):
        h, dy, dres, w = (rows(r, c, H, k) for k in range(4))
        w = w[0].clone()
        dx, dw = grad(dy, h, w, dres)
        for _ in range(3):  # sums in a fixed order
            again = grad(dy, h, w, dres)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
        for over in range(3):
            ins = [dy.clone(), h.clone(), dres.clone()]
            got = grad(ins[0], ins[1], w, ins[2], dx=ins[over])
            assert torch.equal(got[0], dx) and torch.equal(got[1], dw)


@pytest.mark.gpu
def test_nothing_to_norm(dev):
    e = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    norm(e(0, 64), e(64), fmt=0)
    norm(e(5, 0), e(0), fmt=0)
    dx, dw = grad(e(0, 64), e(0, 64), e(64))
    assert (dw == 0).all()
    grad(e(5, 0), e(5, 0), e(0))


@pytest.mark.gpu
def test_types_and_devices_are_refused(dev):
    x, w = rows(4, 64, F, 1), rows(1, 64, F, 2)[0]
    y = torch.empty_like(x)
    go = lambda *b, kind=0, wkind=0: M.launch(M.kernels.rms_norm, (*b, 64, kind, wkind, 0, 0, 1e-6), 4, stream=stream())  # noqa: E731
    for args, kw, match in (((y, None, None, None, x.to(H), None, w), {}, "expected Float32"),
                            ((y, None, None, None, x, None, w.to(H)), {}, "expected Float32"),
                            ((y, None, None, None, x, None, w), {"wkind": 1}, "expected bfloat16"),
                            ((y.to(H), None, None, None, x.to(H), None, w), {}, "expected Float32"),
                            ((y, None, None, None, x.t().contiguous().t(), None, w), {}, "contiguous"),
                            ((y, None, None, None, x.cpu(), None, w), {}, "current device"),
                            ((y, torch.empty((4, 64), dtype=torch.float8_e5m2, device="cuda"), w, None, x, None, w), {}, "expected 8-bit codes in e4m3")):
        with pytest.raises(M.ArgumentError, match=match):
            go(*args, **kw)
    with pytest.raises(M.ArgumentError, match="scratch"):
        M.launch(M.kernels.rms_norm_grad, (y, torch.empty_like(w), x, x, w, None, 64, 0, 0, 1e-6), 4, stream=stream(),
                 workspace=torch.empty(1 << 20))


@pytest.mark.gpu
def test_captured_on_other_streams_and_in_a_graph(dev):
    r, c = 300, 1160
    x, res, w, dy = rows(r, c, H, 1), rows(r, c, H, 2), rows(1, c, F, 3)[0], rows(r, c, H, 4)
    y, h, q, s = norm(x, w, res, fmt=0)
    dx, dw = grad(dy, h, w, dy)
    # captured, and replayed on new inputs in the same places
    y1, h1, q1, s1 = (torch.zeros_like(v) for v in (y, h, q.view(torch.uint8), s))
    dx1, dw1 = torch.zeros_like(dx), torch.zeros_like(dw)
    x1, res1 = torch.zeros_like(x), torch.zeros_like(res)
    args = (dx1, dw1, dy, h1, w, dy, c, 1, 0, 1e-6)
    scratch = torch.empty(M.workspace_bytes(M.kernels.rms_norm_grad, args, r), dtype=torch.uint8, device="cuda")
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        M.launch(M.kernels.rms_norm, (y1, q1, s1, h1, x1, res1, w, c, 1, 0, 0, 0, 1e-6), r, stream=stream())
        M.launch(M.kernels.rms_norm_grad, args, r, stream=stream(), workspace=scratch)
    x1.copy_(x)
    res1.copy_(res)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b in ((y1, y), (h1, h), (q1, q.view(torch.uint8)), (s1, s), (dx1, dx), (dw1, dw)):
        assert torch.equal(a, b)
    # as passes of a plan, whose scratch is the plan's own
    B = lambda t, d: M.Buffer.wrap(dev, t, dtype=d)  # noqa: E731
    X, RES, DY, Wt = B(x, np.uint16), B(res, np.uint16), B(dy, np.uint16), B(w, np.float32)
    Hb, DX, DW = M.Buffer(dev, np.uint16, r * c), M.Buffer(dev, np.uint16, r * c), M.Buffer(dev, np.float32, c)
    Y = M.Buffer(dev, np.uint16, r * c)
    G = M.Graph(dev)
    R, Wr = (lambda p, b: M.use(p, b, read=True)), (lambda p, b: M.use(p, b, write=True))
    M.compute(G, "norm", lambda p: M.dispatch(p, M.kernels.rms_norm, (
        Wr(p, Y), None, None, Wr(p, Hb), R(p, X), R(p, RES), R(p, Wt), c, 1, 0, 0, 0, 1e-6), r))
    M.compute(G, "grad", lambda p: M.dispatch(p, M.kernels.rms_norm_grad, (
        Wr(p, DX), Wr(p, DW), R(p, DY), R(p, Hb), R(p, Wt), R(p, DY), c, 1, 0, 1e-6), r))
    plan = M.Plan(G)
    for _ in range(2):
        M.run(plan)
    dev.synchronize()
    bits = lambda t: t.view(torch.int16).cpu().numpy().view(np.uint16).reshape(-1)  # noqa: E731
    # a plan of the gradient alone, which is two kernels
    H2, DX2, DW2, G2 = B(h, np.uint16), M.Buffer(dev, np.uint16, r * c), M.Buffer(dev, np.float32, c), M.Graph(dev)
    M.compute(G2, "grad", lambda p: M.dispatch(p, M.kernels.rms_norm_grad, (
        Wr(p, DX2), Wr(p, DW2), R(p, DY), R(p, H2), R(p, Wt), R(p, DY), c, 1, 0, 1e-6), r))
    alone = M.Plan(G2)
    for _ in range(3):
        M.run(alone)
        M.run(plan)
    dev.synchronize()
    assert np.array_equal(DX2.array(), bits(dx)) and np.array_equal(DW2.array(), dw.cpu().numpy())
    assert np.array_equal(Y.array(), bits(y)) and np.array_equal(DX.array(), bits(dx)) and np.array_equal(DW.array(), dw.cpu().numpy())


@pytest.mark.gpu
def test_norm_past_2_to_the_31_values(dev):
    r, c = 2_100_000, 1032
    x = torch.zeros((r, c), dtype=H, device="cuda")
    x[-3:] = rows(3, c, H, 1)
    w = rows(1, c, F, 2)[0]
    M.launch(M.kernels.rms_norm, (x, None, None, None, x, None, w, c, 1, 0, 0, 0, 1e-6), r, stream=stream())
    torch.cuda.synchronize()
    check_y(x[-3:], exact(rows(3, c, H, 1), w)[1])
