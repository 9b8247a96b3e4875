"""The bf16 products grouped by expert and their gradients against 64-bit arithmetic.

Tolerance: the products of bf16 values are exact in fp32; an MMA adds 16 of them to
the running sum, each addition off by at most one unit of fp32 (2^-23) of a partial
sum that S = sum |a b| bounds: |out - exact| <= (D + 16) * 2^-23 * S over D terms, and
a bf16 output adds half a step, 2^-8 of the value. fp32 outputs are also held to a
relative Frobenius error of 1e-5, the bound of the dense GEMM's tests.
"""
import pytest
import torch

import mantle_cuda as M

ptr = lambda n, at=1 << 20: M.DevicePtr(at, n)  # noqa: E731


def args(way, e, t, n, k, out=0, **change):
    w, x, y = e * k * n, t * k, t * n
    c, a, b = {"fwd": (y, x, w), "dx": (x, y, w), "dw": (w, x, y)}[way]
    z = dict(c=c * (2 if out == 1 else 4), a=a * 2, b=b * 2, off=4 * (e + 1)) | change
    return [ptr(z["c"]), ptr(z["a"]), ptr(z["b"]), ptr(z["off"]), t, n, k, out]


KERNEL = {"fwd": "gemm_grouped_bf16", "dx": "gemm_grouped_dx_bf16", "dw": "gemm_grouped_dw_bf16"}
WAYS = list(KERNEL)


@pytest.mark.parametrize("way", WAYS)
def test_refusals(way):
    k = getattr(M.kernels, KERNEL[way])
    for a, e, match in [
        (args(way, 3, 10, 40, 24, out=2), 3, "output type"),
        (args(way, 3, 10, 44, 24), 3, "multiples of 8"),
        (args(way, 3, 10, 40, 20), 3, "multiples of 8"),
        (args(way, 3, -1, 40, 24), 3, "negative"),
        (args(way, 3, 10, 40, 24, off=12), 3, "offsets"),
        (args(way, 1100, 10, 40, 24), 1100, "more than 1024 groups"),
    ]:
        with pytest.raises(M.MantleError, match=match):
            M.launch(k, a, e)
    for i, which in enumerate("cab"):
        full = args(way, 3, 10, 40, 24)[i].nbytes
        with pytest.raises(M.MantleError, match="the launch touches"):
            M.launch(k, args(way, 3, 10, 40, 24, **{which: full - 1}), 3)
    bad = args(way, 3, 10, 40, 24)
    bad[1] = M.DevicePtr((1 << 20) + 2, 1 << 20)
    with pytest.raises(M.MantleError, match="16-byte aligned"):
        M.launch(k, bad, 3)
    with pytest.raises(M.ArgumentError, match="contiguous CUDA tensor"):
        M.launch(k, [torch.zeros(400)] + args(way, 3, 10, 40, 24)[1:], 3)
    if way != "dw":
        zero = args(way, 3, 10, 40, 0) if way == "fwd" else args(way, 3, 10, 0, 24)
        with pytest.raises(M.MantleError, match="contraction"):
            M.launch(k, zero, 3)


# ── on the GPU ───────────────────────────────────────────────────────────────
def normal(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(torch.bfloat16)


def launch(way, out, a, b, offsets, t, n, k, e, kind):
    M.launch(getattr(M.kernels, KERNEL[way]), (out, a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), t, n, k, kind), e,
             stream=torch.cuda.current_stream().cuda_stream)


def check(got, a, b, kind):
    """got against a @ b (float64 operands)."""
    want, total = a @ b, a.abs() @ b.abs()
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    tol = (a.shape[1] + 16) * 2.0 ** -23 * total + (2.0 ** -8 * want.abs() if kind else 0.0)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    if not kind and want.numel():
        assert (got - want).norm() <= 1e-5 * want.norm()


SIZES = [
    ([1], 0, 1, 8, 8),
    ([3, 0, 1, 16], 0, 20, 72, 200),
    ([5, 130, 0, 64, 1, 17], 3, 230, 264, 136),     # rows before the first and behind the last group
    ([128, 256, 127, 129], 0, 640, 512, 264),
    ([700, 20, 600], 0, 1320, 520, 1000),
    ([2] * 40, 0, 80, 640, 512),
    ([0, 0, 0], 0, 5, 64, 64),
    ([1000, 1100], 0, 2100, 2056, 1032),
    ([300] * 6 + [0, 31], 0, 1831, 1024, 648),
    # many groups of a few rows (rows as the MMA's N operand, 32 or 64 of them), some of more than a tile has
    ([1, 0, 33, 5, 0, 2, 70, 16, 1, 1] * 3, 5, 400, 1032, 1000),
    ([0, 9, 15, 0, 31, 32, 1] * 6, 0, 530, 640, 584),
    ([20, 0, 65, 128, 3, 30, 31, 1] * 4, 2, 1120, 1024, 1096),
    # large groups, enough 256 x 256 tiles for CTA pairs in every form; chunked and ragged widths
    ([2500, 0, 1800, 700], 3, 5010, 2056, 2104),
    ([3001, 1999], 0, 5000, 2112, 1984),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("sizes,first,t,n,k", SIZES)
def test_forward_and_gradients(dev, sizes, first, t, n, k, kind):
    e = len(sizes)
    o = [first + sum(sizes[:i]) for i in range(e + 1)]
    x, dy, w = normal((t, k), t + k), normal((t, n), t + n), normal((e, k, n), n + k)
    dt = torch.bfloat16 if kind else torch.float32
    xg, dyg, wg = x.cuda(), dy.cuda(), w.cuda()
    y = torch.full((t, n), 3.0, dtype=dt, device="cuda")
    dx = torch.full((t, k), 3.0, dtype=dt, device="cuda")
    dw = torch.full((e, k, n), float("nan"), dtype=dt, device="cuda")
    launch("fwd", y, xg, wg, o, t, n, k, e, kind)
    launch("dx", dx, dyg, wg, o, t, n, k, e, kind)
    launch("dw", dw, xg, dyg, o, t, n, k, e, kind)
    torch.cuda.synchronize()
    x, dy, w = x.double(), dy.double(), w.double()
    for i in range(e):
        r = slice(o[i], o[i + 1])
        check(y[r], x[r], w[i], kind)
        check(dx[r], dy[r], w[i].t(), kind)
        check(dw[i], x[r].t(), dy[r], kind)
    for v in (y, dx):
        assert (v[:o[0]] == 3.0).all() and (v[o[-1]:] == 3.0).all()
    assert M.kernel_timeouts() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_other_groups_rows_do_not_reach_a_group(dev, way):
    # groups 0 and 2 and the rows of no group hold NaN and infinities; group 1's results stay exact
    sizes, t, n, k = [37, 45, 50], 140, 136, 200
    o = [4, 41, 86, 136]
    x, dy, w = normal((t, k), 1), normal((t, n), 2), normal((3, k, n), 3)
    for v in (x, dy):
        v[:41] = float("nan")
        v[86:] = float("inf")
    w[0], w[2] = float("nan"), float("nan")
    out = torch.zeros({"fwd": (t, n), "dx": (t, k), "dw": (3, k, n)}[way], device="cuda")
    a, b = {"fwd": (x, w), "dx": (dy, w), "dw": (x, dy)}[way]
    launch(way, out, a.cuda(), b.cuda(), o, t, n, k, 3, 0)
    torch.cuda.synchronize()
    r = slice(41, 86)
    x, dy, w = x.double(), dy.double(), w.double()
    if way == "dw":
        check(out[1], x[r].t(), dy[r], 0)
    else:
        check(out[r], *((x[r], w[1]) if way == "fwd" else (dy[r], w[1].t())), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(520, 264), (576, 320)])
def test_other_groups_rows_do_not_reach_a_weight_gradient_of_many_groups(dev, k, n):
    # enough tiles for CTA pairs; every other group and the rows of no group hold NaN and infinities
    sizes = [(7 * i) % 131 for i in range(40)]
    o = [4 + sum(sizes[:i]) for i in range(41)]
    t = o[-1] + 9
    x, dy = normal((t, k), 1), normal((t, n), 2)
    bad = torch.ones(t, dtype=torch.bool)
    for i in range(1, 40, 2):
        bad[o[i]:o[i + 1]] = False
    for v in (x, dy):
        v[bad] = float("nan")
        v[:2] = float("inf")
    out = torch.full((40, k, n), 7.0, device="cuda")
    launch("dw", out, x.cuda(), dy.cuda(), o, t, n, k, 40, 0)
    torch.cuda.synchronize()
    x, dy = x.double(), dy.double()
    for i in range(1, 40, 2):
        r = slice(o[i], o[i + 1])
        check(out[i], x[r].t(), dy[r], 0)
    for i in range(40):
        if sizes[i] == 0:
            assert float(out[i].abs().max()) == 0.0


@pytest.mark.gpu
def test_rows_behind_a_group_stay_out_of_its_weight_gradient_every_time(dev):
    # Groups of every length modulo 64 on CTA pairs, each CTA clearing its own half of a group's last rows. Groups of NaN
    # lie between them and fill shared memory before and after; one launch that took a row uncleared would show it.
    k, n = 320, 328
    sizes = [m for i in range(64) for m in (64 + i, 70)]
    o = [sum(sizes[:i]) for i in range(129)]
    t = o[-1]
    x, dy = normal((t, k), 5).cuda(), normal((t, n), 6).cuda()
    for i in range(1, 128, 2):
        x[o[i]:o[i + 1]], dy[o[i]:o[i + 1]] = float("nan"), float("inf")
    out = torch.full((2, 128, k, n), 7.0, device="cuda")
    for i in range(200):
        launch("dw", out[int(i > 0)], x, dy, o, t, n, k, 128, 0)
        if i:
            assert torch.equal(out[0, ::2], out[1, ::2]), i
    for i in range(0, 128, 2):
        r = slice(o[i], o[i + 1])
        check(out[0, i], x[r].double().cpu().t(), dy[r].double().cpu(), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_bad_offsets_stay_in_bounds(dev, way):
    t, n, k = 100, 136, 72
    x, dy, w = normal((t, k), 1).cuda(), normal((t, n), 2).cuda(), normal((4, k, n), 3).cuda()
    off = [-5, 40, 20, 90, 1 << 30]  # clamped: 0..40, none, 40..90, 90..100
    rows = {"fwd": (t, n), "dx": (t, k), "dw": (4 * k, n)}[way]
    guard = torch.full((rows[0] + 64, rows[1]), 3.0, device="cuda")
    a, b = {"fwd": (x, w), "dx": (dy, w), "dw": (x, dy)}[way]
    launch(way, guard[:rows[0]], a, b, off, t, n, k, 4, 0)
    torch.cuda.synchronize()
    assert (guard[rows[0]:] == 3.0).all() and torch.isfinite(guard).all()
    x, dy, w, got = x.double().cpu(), dy.double().cpu(), w.double().cpu(), guard.double().cpu()
    for e, lo, hi in ((0, 0, 20), (0, 0, 40), (1, 40, 40), (2, 40, 90), (3, 90, 100)):
        if way == "dw":
            if (lo, hi) != (0, 20):
                check(got[e * k:(e + 1) * k], x[lo:hi].t(), dy[lo:hi], 0)
        else:
            check(got[lo:hi], *((x[lo:hi], w[e]) if way == "fwd" else (dy[lo:hi], w[e].t())), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("t", [100, 1600])
def test_offsets_that_fall_give_no_row_to_two_groups(dev, way, t):
    # 0, T, 0, T, ...: the first group has every row, the others none; with 100 rows as the MMA's N operand
    e, n, k = 32, 1032, 1000
    x, dy, w = normal((t, k), 1).cuda(), normal((t, n), 2).cuda(), normal((e, k, n), 3).cuda()
    out = torch.full({"fwd": (t, n), "dx": (t, k), "dw": (e, k, n)}[way], 3.0, device="cuda")
    a, b = {"fwd": (x, w), "dx": (dy, w), "dw": (x, dy)}[way]
    launch(way, out, a, b, [0, t] * (e // 2) + [0], t, n, k, e, 0)
    torch.cuda.synchronize()
    x, dy, w = x.double().cpu(), dy.double().cpu(), w[0].double().cpu()
    if way == "dw":
        check(out[0], x.t(), dy, 0)
        assert float(out[1:].abs().max()) == 0.0
    else:
        check(out, *((x, w) if way == "fwd" else (dy, w.t())), 0)
    assert M.kernel_timeouts() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("way,sizes,n,k", [
    ("fwd", [200], 136, 8192), ("dx", [200], 8192, 136), ("dw", [8200], 136, 200),      # one CTA a tile, 128 columns
    ("fwd", [300] * 4, 2048, 4100 // 8 * 8), ("dw", [4100] * 20, 264, 200),               # 256 columns, and pairs
    ("fwd", [2] * 40, 1024, 8192), ("dx", [33, 0, 5] * 14, 8192, 1032),                  # rows as the MMA's N operand
    ("fwd", [2600, 2520], 1024, 8192), ("dx", [2600, 2520], 8192, 1024), ("dw", [8192, 8200], 1792, 1800),  # CTA pairs
])
def test_long_contractions_in_fp32(dev, way, sizes, n, k):
    # An MMA of 16 products is off by up to 2^-23 of the sum it adds to. With terms of one size the sum after j MMAs
    # is of size 4 sqrt(j), so the 48 of a run of 768 terms are off by sum 4 sqrt(j) 2^-23 = 900 * 2^-23 where its
    # own size is sqrt(768): 32.5 * 2^-23 = 3.9e-6 of it at most, if all errors point one way. Runs are added with
    # half a unit of rounding each, 11 of them 11 * 2^-24 = 0.7e-6 at most: 4.6e-6 in all, whatever the length. (One
    # accumulator over 8192 terms may be off by ten times the first part, and is by 8e-6.)
    e, t = len(sizes), sum(sizes)
    o = [sum(sizes[:i]) for i in range(e + 1)]
    g = torch.Generator(device="cuda").manual_seed(n + k)
    a, b = ({"fwd": (t, k), "dx": (t, n), "dw": (t, k)}[way], {"fwd": (e, k, n), "dx": (e, k, n), "dw": (t, n)}[way])
    a, b = (torch.randn(v, generator=g, device="cuda").to(torch.bfloat16) for v in (a, b))
    out = torch.full({"fwd": (t, n), "dx": (t, k), "dw": (e, k, n)}[way], float("nan"), device="cuda")
    launch(way, out, a, b, o, t, n, k, e, 0)
    for i in range(e):
        r = slice(o[i], o[i + 1])
        if sizes[i] == 0:
            continue
        x, y = (a[r].double().t(), b[r].double()) if way == "dw" else (a[r].double(), b[i].double().t() if way == "dx" else b[i].double())
        want = x @ y
        off = (out[i] if way == "dw" else out[r]).double() - want
        assert float(off.norm()) <= 4.6e-6 * float(want.norm())
    assert M.kernel_timeouts() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,n,k", [
    ([8192] + [0] * 15, 136, 200), ([12000] + [8] * 63, 136, 136),     # one CTA a tile
    ([8192] + [0] * 15, 1792, 1800), ([12000] + [8] * 63, 520, 264),   # pairs, groups short on average
    ([9000] + [100] * 15, 1800, 1800),                                  # pairs, longer ones
    # a run and a little more or less, long groups between short and empty ones
    ([700, 768, 769, 0, 5000, 832, 64, 1, 1536, 1537, 0, 767], 264, 200),
    ([700, 768, 769, 0, 5000, 832, 64, 1, 1536, 1537, 0, 767], 776, 1032),
    ([900, 0, 3] * 40, 264, 136),
])
def test_a_weight_gradients_long_groups_among_short_ones_in_fp32(dev, sizes, n, k):
    # The bound of the test above, 3.9e-6 for a run of 768 terms and half a unit of rounding for each run that is
    # added, for every group by its own length, whatever the others'. Groups of up to 16 rows are left to the bound of
    # `check`: over few elements errors do not add up as the bound's root of the terms.
    e, t = len(sizes), sum(sizes)
    o = [sum(sizes[:i]) for i in range(e + 1)]
    g = torch.Generator(device="cuda").manual_seed(n + k + e)
    x, dy = (torch.randn(v, generator=g, device="cuda").to(torch.bfloat16) for v in ((t, k), (t, n)))
    out = torch.full((2, e, k, n), float("nan"), device="cuda")
    for i in range(2):
        launch("dw", out[i], x, dy, o, t, n, k, e, 0)
    assert torch.equal(out[0], out[1])
    for i in range(e):
        r = slice(o[i], o[i + 1])
        a, b = x[r].double().t(), dy[r].double()
        want = a @ b
        if sizes[i] <= 16:
            assert ((out[0, i].double() - want).abs() <= (sizes[i] + 16) * 2.0 ** -23 * (a.abs() @ b.abs())).all()
        else:
            runs = -(-sizes[i] // 768)
            assert float((out[0, i].double() - want).norm()) <= (3.9e-6 + runs * 2.0 ** -24) * float(want.norm()), sizes[i]
    assert M.kernel_timeouts() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("way,sizes,n,k", [
    ("dw", [8_000_000], 16, 16), ("fwd", [16], 16, 8_000_000), ("dx", [16], 8_000_000, 16),  # one CTA a tile
    ("dw", [3_000_000, 40, 32768, 0, 32769], 136, 72), ("fwd", [500] * 4, 2560, 40_000),
    ("dw", [1_000_000, 5, 40_000], 1288, 1032), ("dw", [33_000] + [35] * 200, 264, 136), ("fwd", [5120], 1024, 40_000), ("dx", [5120], 40_000, 1024),  # pairs
    ("fwd", [2] * 40, 1024, 40_000),                                                         # few rows a group
])
def test_very_long_contractions_in_bf16(dev, way, sizes, n, k):
    # Sums of more than 32768 terms are added run by run. As above, the 2048 MMAs of a run are off by sum 4 sqrt(j) 2^-23
    # = 2.5e5 * 2^-23 at most where the run's own size is 181: 1.63e-4 of it. Runs are added with half a unit of fp32
    # each, and the result is rounded to bf16: 2^-8 of the value. No wait takes as long as the sum: the limit is 10 ms
    # here, and the 8 million terms of a tile take longer.
    e, t = len(sizes), sum(sizes)
    o = [sum(sizes[:i]) for i in range(e + 1)]
    g = torch.Generator(device="cuda").manual_seed(n + k)
    a, b = ({"fwd": (t, k), "dx": (t, n), "dw": (t, k)}[way], {"fwd": (e, k, n), "dx": (e, k, n), "dw": (t, n)}[way])
    a, b = (torch.randn(v, generator=g, device="cuda", dtype=torch.bfloat16) for v in (a, b))
    out = torch.full({"fwd": (t, n), "dx": (t, k), "dw": (e, k, n)}[way], float("nan"), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    try:
        M.set_wait_limit(10_000_000)
        launch(way, out, a, b, o, t, n, k, e, 1)
        torch.cuda.synchronize()
    finally:
        M.set_wait_limit(0)
    assert M.kernel_timeouts(reset=True) == 0
    for i in range(e):
        r = slice(o[i], o[i + 1])
        x, y = (a[r].t(), b[r]) if way == "dw" else (a[r], b[i].t() if way == "dx" else b[i])
        want = torch.zeros((x.shape[0], y.shape[1]), dtype=torch.float64, device="cuda")
        for c in range(0, x.shape[1], 1 << 18):
            want += x[:, c:c + (1 << 18)].double() @ y[c:c + (1 << 18)].double()
        off = (out[i] if way == "dw" else out[r]).double() - want
        assert float(off.norm()) <= (2.0 ** -8 + 1.63e-4 + -(-x.shape[1] // 32768) * 2.0 ** -24) * float(want.norm())


@pytest.mark.gpu
def test_the_gradients_are_the_products_derivatives(dev):
    # the directional derivative of L = sum(Y * dY) by central differences: L is linear in X and in W, so a step
    # of h along a direction D changes L by h <grad, D> exactly, up to the sums' rounding (fp32, S as above) and
    # the rounding of X + h D to bf16, which is avoided by taking steps that bf16 holds exactly
    sizes, t, n, k, h = [33, 0, 70], 103, 64, 72, 1.0
    o = [0, 33, 33, 103]
    g = torch.Generator().manual_seed(4)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    x, w, dy, dirx, dirw = whole(t, k), whole(3, k, n), whole(t, n), whole(t, k), whole(3, k, n)

    def loss(xv, wv):
        y = torch.zeros((t, n), device="cuda")
        launch("fwd", y, xv, wv, o, t, n, k, 3, 0)
        return (y.double() * dy.double()).sum()

    dx, dw = torch.zeros((t, k), device="cuda"), torch.zeros((3, k, n), device="cuda")
    launch("dx", dx, dy, w, o, t, n, k, 3, 0)
    launch("dw", dw, x, dy, o, t, n, k, 3, 0)
    # whole numbers below 2^24 throughout: every product and sum is exact
    assert float((loss(x + h * dirx, w) - loss(x - h * dirx, w)) / (2 * h)) == float((dx.double() * dirx.double()).sum())
    assert float((loss(x, w + h * dirw) - loss(x, w - h * dirw)) / (2 * h)) == float((dw.double() * dirw.double()).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1])
def test_weight_gradients_of_a_thousand_groups(dev, kind):
    # as many groups as there may be, two of them of several runs, among empty ones; whole numbers: exact in fp32
    e, k, n = 1024, 64, 72
    sizes = [i % 4 for i in range(e)]
    sizes[5], sizes[1023] = 900, 2000
    o = [sum(sizes[:i]) for i in range(e + 1)]
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randint(-3, 4, s, generator=g).to(torch.bfloat16) for s in ((o[-1], k), (o[-1], n)))
    out = torch.full((e, k, n), float("nan"), dtype=torch.bfloat16 if kind else torch.float32, device="cuda")
    launch("dw", out, x.cuda(), dy.cuda(), o, o[-1], n, k, e, kind)
    torch.cuda.synchronize()
    for i in range(e):
        want = x[o[i]:o[i + 1]].float().t() @ dy[o[i]:o[i + 1]].float()
        assert torch.equal(out[i].cpu(), want.to(out.dtype)), i
