"""The experts' rows back to their tokens, and the gradient, against 64-bit arithmetic.

u = 2^-24. A value of y is a chain of `top` fused products and the base's addition: off by
(top + 1) u of sum |w v| + |base|, and half a step of its type. A row's gradient is one
product, u, and half a step. A weight's gradient sums C products: a thread's eight a tile
of columns, ten levels of a tree, and a tile each: (18 + tiles) u of sum |dy v|, where a
tile has 1024 columns or more.
"""
import numpy as np
import pytest
import torch

import mantle_cuda as M
from mantle_cuda.workloads import build_moe, rows_of_codes

u = 2.0 ** -24
F, H = torch.float32, torch.bfloat16
HALF = {F: u, H: 2.0 ** -8}
ptr = lambda n, at=1 << 20: M.DevicePtr(at, n)  # noqa: E731


# ── refusals (no launch) ─────────────────────────────────────────────────────
def c_args(t=4, R=8, c=100, top=2, kind=0, ykind=0, **change):
    per, pery = (2 if k == 1 else 4 for k in (kind, ykind))
    a = dict(y=ptr(t * c * pery), rows=ptr(R * c * per), w=ptr(4 * t * top), at=ptr(4 * t * top), base=None)
    a.update(change)
    return [*a.values(), R, c, top, kind, ykind]


@pytest.mark.parametrize("args,nd,match", [
    (c_args(y=ptr(1599)), 4, "y: 1599"), (c_args(rows=ptr(3199)), 4, "the rows"), (c_args(w=ptr(31)), 4, "the weights"),
    (c_args(at=ptr(31)), 4, "row_at"), (c_args(base=ptr(1599)), 4, "base"), (c_args(), 5, "y: 1600"), (c_args(R=9, rows=ptr(3200)), 4, "the rows"),
    (c_args(top=0), 4, "top must be"), (c_args(top=33), 4, "top must be"), (c_args(R=-1), 4, "negative"), (c_args(c=-1), 4, "negative"),
    (c_args(kind=2), 4, "must be 0 or 1"), (c_args(ykind=2), 4, "must be 0 or 1"), (c_args(), (4, 2), "one-dimensional"),
    (c_args(rows=ptr(1 << 20, (1 << 20) + 2)), 4, "4-byte aligned"), (c_args(rows=ptr(0, 0)), 4, "the rows must be a device buffer"),
    (c_args(w=ptr(0, 0)), 4, "the weights must be a device buffer"), (c_args(base=ptr(0, 0)), 4, "base must be a device buffer"),
])
def test_combine_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.combine_experts, args, nd)


def d_args(t=4, R=8, c=100, top=2, kind=0, ykind=0, **change):
    per, pery = (2 if k == 1 else 4 for k in (kind, ykind))
    a = dict(drows=ptr(R * c * per), dw=ptr(4 * t * top), dy=ptr(t * c * pery), rows=ptr(R * c * per), w=ptr(4 * t * top), at=ptr(4 * t * top), of=ptr(4 * R))
    a.update(change)
    return [*a.values(), R, c, top, kind, ykind]


@pytest.mark.parametrize("args,nd,match", [
    (d_args(drows=ptr(3199)), 4, "drows"), (d_args(dw=ptr(31)), 4, "the weights' gradient"), (d_args(dy=ptr(1599)), 4, "dy"),
    (d_args(rows=ptr(3199)), 4, "the rows"), (d_args(w=ptr(31)), 4, "the weights"), (d_args(at=ptr(31)), 4, "row_at"),
    (d_args(of=ptr(31)), 4, "rows_of"), (d_args(rows=None), 4, "needs the rows"), (d_args(), 5, "the weights' gradient"),
    (d_args(top=33), 4, "top must be"), (d_args(kind=2), 4, "must be 0 or 1"), (d_args(ykind=-2), 4, "must be 0 or 1"),
    (d_args(of=ptr(0, 0)), 4, "rows_of must be a device buffer"),
])
def test_combine_grad_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.combine_experts_grad, args, nd)


# ── on the device ────────────────────────────────────────────────────────────
def stream():
    return torch.cuda.current_stream().cuda_stream


def values(shape, kind, seed, at=0):
    n = int(np.prod(shape))
    return torch.randn(n + at, generator=torch.Generator().manual_seed(seed)).to(kind).cuda()[at:].view(shape)


def places(t, top, seed, dropped=0.0):
    """(row_at (t, top), rows_of) of a random order of the slots, some without a row."""
    g = torch.Generator().manual_seed(seed)
    n = t * top
    has = torch.rand(n, generator=g) >= dropped
    rows = int(has.sum())
    at = torch.full((n,), -1, dtype=torch.int32)
    at[has] = torch.randperm(rows, generator=g).to(torch.int32)
    of = torch.full((n,), -1, dtype=torch.int32)
    of[at[has].long()] = (torch.arange(n)[has] // top).to(torch.int32)
    return at.view(t, top).cuda(), of.cuda()


def combine(rows, w, at, base, c, ykind, out=None):
    t, top = at.shape
    y = torch.full((t, c), float("nan"), dtype=ykind, device="cuda") if out is None else out
    M.launch(M.kernels.combine_experts, (y, rows, w, at, base, rows.shape[0], c, top, int(rows.dtype == H), int(ykind == H)), t, stream=stream())
    torch.cuda.synchronize()
    return y


def of_slots(rows, at):
    """(t, top, c) in 64 bits, zeros for a slot without a row."""
    r = torch.cat((rows.double().cpu(), torch.zeros(1, rows.shape[1], dtype=torch.float64)))
    i = at.cpu().long()
    return r[torch.where((i < 0) | (i >= rows.shape[0]), rows.shape[0], i)]


SHAPES = [(1, 1, 1), (1, 2, 2048), (3, 2, 8), (7, 3, 100), (5, 8, 264), (4, 4, 1024), (6, 2, 1032), (3, 5, 1999), (2, 8, 2056), (3, 6, 4096), (1, 32, 5000), (300, 2, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,ykind", [(F, F), (H, H), (H, F), (F, H)])
@pytest.mark.parametrize("t,top,c", SHAPES)
def test_combine(dev, t, top, c, kind, ykind):
    for off in (0, 1):
        for dropped in (0.0, 0.4, 1.0):
            at, _ = places(t, top, t, dropped)
            rows, w, base = values((t * top, c), kind, 1, off), values((t, top), F, 2), values((t, c), ykind, 3, off)
            v = of_slots(rows, at)
            for weight, b in ((w, base), (w, None), (None, None)):
                y = combine(rows, weight, at, b, c, ykind)
                terms = v * (1.0 if weight is None else weight.double().cpu()[:, :, None])
                b64 = torch.zeros(t, c, dtype=torch.float64) if b is None else b.double().cpu()
                want, mag = terms.sum(1) + b64, terms.abs().sum(1) + b64.abs()
                tol = (top + 1) * u * mag
                assert ((y.double().cpu() - want).abs() <= tol + HALF[ykind] * (want.abs() + tol)).all()
    # on top of the base itself
    y = combine(rows, w, at, base, c, ykind)
    over = base.clone()
    assert torch.equal(combine(rows, w, at, over, c, ykind, out=over), y)


@pytest.mark.gpu
def test_rows_outside_and_weights_that_are_not_numbers(dev):
    rows, w = values((6, 40), F, 1), values((3, 2), F, 2)
    at = torch.tensor([[0, 6], [-5, 2 ** 31 - 1], [-2 ** 31, 5]], dtype=torch.int32, device="cuda")
    y = combine(rows, w, at, None, 40, F)
    assert torch.equal(y[0], rows[0] * w[0, 0]) and (y[1] == 0).all() and torch.equal(y[2], rows[5] * w[2, 1])
    w[1, 0] = float("nan")  # as of a token whose logits are not numbers: its row says so
    rows[3] = float("nan")  # no slot's row
    y = combine(rows, w, at, None, 40, F)
    assert y[1].isnan().all() and not y[[0, 2]].isnan().any()


def grad(dy, rows, w, at, of, dw=True, kind=None, drows=None):
    t, top = at.shape
    R, c = (of.numel(), dy.shape[1])
    kind = rows.dtype if rows is not None else kind
    drows = torch.full((R, c), 7.0, dtype=kind, device="cuda") if drows is None else drows
    dw = torch.full((t, top), float("nan"), device="cuda") if dw else None
    M.launch(M.kernels.combine_experts_grad, (drows, dw, dy, rows, w, at, of, R, c, top, int(kind == H), int(dy.dtype == H)), t, stream=stream())
    torch.cuda.synchronize()
    return drows, dw


@pytest.mark.gpu
@pytest.mark.parametrize("kind,ykind", [(F, F), (H, H), (H, F), (F, H)])
@pytest.mark.parametrize("t,top,c", SHAPES + [(2, 3, 9000)])
def test_combine_grad(dev, t, top, c, kind, ykind):
    for off in (0, 1):
        for dropped in (0.0, 0.4, 1.0):
            at, of = places(t, top, t, dropped)
            rows, w, dy = values((t * top, c), kind, 1, off), values((t, top), F, 2), values((t, c), ykind, 3, off)
            drows, dw = grad(dy, rows, w, at, of)
            G = dy.double().cpu()
            n = int((of >= 0).sum())
            want = torch.zeros(n, c, dtype=torch.float64)
            slot = at.cpu().reshape(-1)
            live = slot >= 0
            want[slot[live].long()] = (G[:, None] * w.double().cpu()[:, :, None]).reshape(-1, c)[live]
            got = drows.double().cpu()
            assert ((got[:n] - want).abs() <= (u + HALF[kind] * (1 + u)) * want.abs()).all()
            assert (got[n:] == 7).all()  # rows behind the last stay as they were
            terms = of_slots(rows, at) * G[:, None]
            tol = (18 + -(-c // 1024)) * u * terms.abs().sum(2)
            assert ((dw.double().cpu() - terms.sum(2)).abs() <= tol).all()
            only, none = grad(dy, None, w, at, of, dw=False, kind=kind)
            assert none is None and torch.equal(only, drows)
    # without weights: the rows gathered
    ones, _ = grad(dy, rows, None, at, of)
    assert torch.equal(ones, grad(dy, rows, torch.ones_like(w), at, of)[0])
    again = grad(dy, rows, w, at, of)
    assert torch.equal(again[0], drows) and torch.equal(again[1], dw)


@pytest.mark.gpu
def test_a_row_named_twice_goes_by_its_own_token(dev):
    dy, rows = values((3, 50), F, 1), values((4, 50), F, 2)
    w = torch.tensor([[2.0, 3.0], [5.0, 7.0], [11.0, 13.0]], device="cuda")
    at = torch.tensor([[1, 0], [1, 1], [2, 9]], dtype=torch.int32, device="cuda")
    of = torch.tensor([0, 1, 0, 2], dtype=torch.int32, device="cuda")
    for _ in range(5):
        d, dw = grad(dy, rows, w, at, of)
        assert torch.equal(d[0], 3 * dy[0]) and torch.equal(d[1], 7 * dy[1])
        assert (d[2] == 7).all() and (d[3] == 7).all()  # row 2 is token 0's, which does not name it
        assert dw[2, 1] == 0


@pytest.mark.gpu
def test_combine_grad_against_differences(dev):
    # y is linear in the rows and in the weights: 64-bit differences of any step are exact but for rounding
    t, top, c = 3, 2, 16
    at, of = places(t, top, 1, 0.2)
    rows, w, dy = values((t * top, c), F, 1), values((t, top), F, 2), values((t, c), F, 3)
    drows, dw = grad(dy, rows, w, at, of)
    loss = lambda r, ww: (dy.double().cpu() * (of_slots(r, at) * ww.double().cpu()[:, :, None]).sum(1)).sum().item()  # noqa: E731
    r64, w64 = rows.double(), w.double()
    for i in range(int((of >= 0).sum())):
        for j in range(c):
            up = r64.clone()
            up[i, j] += 1
            assert abs(loss(up, w64) - loss(r64, w64) - drows[i, j].item()) < 1e-6
    for i in range(t):
        for j in range(top):
            up = w64.clone()
            up[i, j] += 1
            assert abs(loss(r64, up) - loss(r64, w64) - dw[i, j].item()) < 1e-5


@pytest.mark.gpu
def test_nothing_to_combine(dev):
    e = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, -1, dtype=torch.int32, device="cuda")  # noqa: E731
    combine(e(0, 64), e(0, 2), i(0, 2), None, 64, F)
    combine(e(6, 0), e(3, 2), i(3, 2), None, 0, F)
    assert (combine(e(0, 64), torch.ones(3, 2, device="cuda"), i(3, 2), None, 64, F) == 0).all()
    grad(e(0, 64), e(6, 64), e(0, 2), i(0, 2), i(6))
    _, dw = grad(e(3, 64), e(0, 64), e(3, 2), i(3, 2), i(0))  # no rows at all
    assert (dw == 0).all()
    _, dw = grad(e(3, 0), e(6, 0), e(3, 2), i(3, 2), i(6))
    assert (dw == 0).all()


@pytest.mark.gpu
def test_captured_and_at_once(dev):
    t, top, c = 500, 3, 1160
    at, of = places(t, top, 1, 0.1)
    rows, w, dy = values((t * top, c), H, 1), values((t, top), F, 2), values((t, c), H, 3)
    want, (drows, dw) = combine(rows, w, at, dy, c, H), grad(dy, rows, w, at, of)
    outs = [(torch.zeros_like(want), torch.full_like(drows, 7.0), torch.zeros_like(dw)) for _ in range(2)]
    graphs, sides = [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for (y, d, e), side in zip(outs, sides):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            M.launch(M.kernels.combine_experts, (y, rows, w, at, dy, t * top, c, top, 1, 1), t, stream=stream())
            M.launch(M.kernels.combine_experts_grad, (d, e, dy, rows, w, at, of, t * top, c, top, 1, 1), t, stream=stream())
        graphs.append(g)
    for _ in range(3):
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for y, d, e in outs:
        assert torch.equal(y, want) and torch.equal(d, drows) and torch.equal(e, dw)


@pytest.mark.gpu
def test_types_and_scratch_are_refused(dev):
    at, of = places(4, 2, 1)
    rows, w, y = values((8, 64), F, 1), values((4, 2), F, 2), torch.empty((4, 64), device="cuda")
    go = lambda *a, kind=0, ykind=0: M.launch(M.kernels.combine_experts, (*a, 8, 64, 2, kind, ykind), 4, stream=stream())  # noqa: E731
    go(y, rows, w, at, None)
    for args, kw, match in (((y, rows.to(H), w, at, None), {}, "expected Float32"), ((y, rows, w, at, None), {"kind": 1}, "expected bfloat16"),
                            ((y, rows, w, at, None), {"ykind": 1}, "expected bfloat16"), ((y, rows, w.to(H), at, None), {}, "expected Float32"),
                            ((y, rows, w, at.long(), None), {}, "expected Int32"), ((y, rows, w, at, y.to(H)), {}, "expected Float32"),
                            ((y, rows.t().contiguous().t(), w, at, None), {}, "contiguous"), ((y, rows, w, at.cpu(), None), {}, "current device")):
        with pytest.raises(M.ArgumentError, match=match):
            go(*args, **kw)


@pytest.mark.gpu
def test_combine_past_2_to_the_31_values(dev):
    R, c = 1_050_000, 2056
    rows = torch.zeros((R, c), dtype=H, device="cuda")
    rows[-1] = 1
    at = torch.tensor([[R - 1, 0], [R, R - 1]], dtype=torch.int32, device="cuda")
    w = torch.tensor([[2.0, 9.0], [9.0, 3.0]], device="cuda")
    y = combine(rows, w, at, None, c, F)
    assert (y[0] == 2).all() and (y[1] == 3).all()
    of = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    of[-1] = 1
    drows, dw = grad(torch.ones((2, c), device="cuda"), rows, w, at, of, drows=torch.zeros_like(rows))
    assert (drows[-1] == 3).all() and dw[0, 0] == c and dw[1, 1] == c and dw[1, 0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top,width,hidden", [(1, 8, 2, 256, 384), (37, 8, 3, 200, 328), (300, 16, 2, 256, 512)])
def test_a_layer_of_experts_routed_on_the_device(dev, tokens, experts, top, width, hidden):
    w = build_moe(dev, tokens, experts, top, width, hidden, seed=3)
    M.run(w.plan)
    first = w.y.array().copy()
    M.run(w.plan)
    assert np.array_equal(w.y.array(), first)
    T, E, eps = tokens * top, experts, 1e-6
    x, scale, router = (w.tensors[n] for n in ("x", "scale", "router"))
    # the same launches outside the graph
    normed = torch.empty_like(x)
    M.launch(M.kernels.rms_norm, (normed, None, None, None, x, None, scale, width, 1, 0, 0, 0, eps), tokens, stream=stream())
    logits = torch.empty((tokens, E), device="cuda")
    M.launch(M.kernels.gemm_bf16, (logits, normed, router, tokens, E, width), 1, stream=stream())
    i = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, rows_of, row_at, off, weights = i(T), i(T), i(T), i(E + 1), torch.empty(T, device="cuda")
    args = (ids, weights, off, rows_of, row_at, logits, None, None, E, top, 1, 1, 1, 0, 1, 0, 1.0)
    need = M.workspace_bytes(M.kernels.route_experts, args, tokens)
    M.launch(M.kernels.route_experts, args, tokens, stream=stream(), workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
    torch.cuda.synchronize()
    for a, b in ((ids, w.ids), (off, w.offsets), (rows_of, w.rows_of), (row_at, w.row_at), (weights, w.routes)):
        assert np.array_equal(a.cpu().numpy(), b.array())
    q = lambda n, m: (torch.empty((n, rows_of_codes(m)), dtype=torch.uint8, device="cuda"), torch.empty((-(-m // 128), n), device="cuda"))  # noqa: E731
    (q1, s1), (q2, s2) = q(T, width), q(T, hidden)
    h, rows = torch.empty((T, hidden), dtype=H, device="cuda"), torch.empty((T, width), dtype=H, device="cuda")
    (up, up_s), (down, down_s) = w.weights["up"], w.weights["down"]
    M.launch(M.kernels.quantize_fp8, (q1, s1, None, None, normed, rows_of, T, width, tokens, 1, 1, 0, 0), 1, stream=stream())
    M.launch(M.kernels.gemm_grouped_fp8, (h, q1, s1, up, up_s, off, T, hidden, width, 0, 0, 1), E, stream=stream())
    M.launch(M.kernels.quantize_fp8, (q2, s2, None, None, h, None, T, hidden, T, 1, 1, 0, 0), 1, stream=stream())
    M.launch(M.kernels.gemm_grouped_fp8, (rows, q2, s2, down, down_s, off, T, width, hidden, 0, 0, 1), E, stream=stream())
    y = combine(rows, weights.view(tokens, top), row_at.view(tokens, top), x, width, H)
    assert np.array_equal(y.view(torch.int16).cpu().numpy().reshape(-1), first.view(np.int16))
    # and the layer before anything was rounded to 8 bits, at the experts chosen: a code is off by 2^-4 of its value at
    # most, five of them (x, both weights, h) and the type's roundings lie on a term's way
    X, W = x.double().cpu(), {n: v.double().cpu() for n, v in w.tensors.items()}
    n64 = X / torch.sqrt((X * X).mean(1, keepdim=True) + eps) * W["scale"]
    l64 = n64 @ W["router"]
    chosen, route = ids.view(tokens, top).cpu().long(), weights.view(tokens, top).double().cpu()
    p = torch.softmax(l64.gather(1, chosen), 1)
    # a logit is off by the roundings of the normalised values to bfloat16 (2^-8) and of their sum
    assert ((route - p).abs() <= 2 * 2.0 ** -7 * (n64.abs() @ W["router"].abs()).amax(1, keepdim=True) * p + 1e-6).all()
    part = torch.stack([torch.stack([W["down"][e] @ (W["up"][e] @ n64[t]) for e in chosen[t]]) for t in range(tokens)])
    want = X + (part * route[:, :, None]).sum(1)
    got = y.double().cpu()
    assert (got - want).norm() <= 0.25 * (want - X).norm()


@pytest.mark.gpu
def test_a_training_step_through_routing_norm_and_experts(dev):
    """Norm, routing, products by expert in bf16 and combination, forward and backward, against
    torch's own differentiation in 64 bits at the same choice of experts. Every value on the way is
    rounded to bfloat16 (2^-8 of itself) a handful of times, so gradients agree to a few hundredths in
    the norm: eight roundings in a row are 8 * 2^-8 = 0.03."""
    T, E, top, C, N = 48, 8, 2, 128, 136
    x, scale, router = values((T, C), H, 1), 1 + 0.1 * values((C,), F, 2), values((C, E), F, 3) / C ** 0.5
    wt, dy = (values((E, C, N), F, 4) / C ** 0.5).to(H), values((T, N), H, 5)
    on = stream()
    normed = torch.empty_like(x)
    M.launch(M.kernels.rms_norm, (normed, None, None, None, x, None, scale, C, 1, 0, 0, 0, 1e-6), T, stream=on)
    logits = normed.float() @ router
    i = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, rows_of, row_at, off, weights = i((T, top)), i(T * top), i((T, top)), i(E + 1), torch.empty((T, top), device="cuda")
    args = (ids, weights, off, rows_of, row_at, logits, None, None, E, top, 1, 1, 1, 0, 1, 0, 1.0)
    M.launch(M.kernels.route_experts, args, T, stream=on)
    xs, rows = torch.empty((T * top, C), dtype=H, device="cuda"), torch.empty((T * top, N), dtype=H, device="cuda")
    M.launch(M.kernels.combine_experts_grad, (xs, None, normed, None, None, row_at, rows_of, T * top, C, top, 1, 1), T, stream=on)
    M.launch(M.kernels.gemm_grouped_bf16, (rows, xs, wt, off, T * top, N, C, 1), E, stream=on)
    y = combine(rows, weights, row_at, None, N, H)
    # backward
    drows, dweights = grad(dy, rows, weights, row_at, rows_of)
    dxs, dwt = torch.empty_like(xs), torch.empty((E, C, N), device="cuda")
    M.launch(M.kernels.gemm_grouped_dx_bf16, (dxs, drows, wt, off, T * top, N, C, 1), E, stream=on)
    M.launch(M.kernels.gemm_grouped_dw_bf16, (dwt, xs, drows, off, T * top, N, C, 0), E, stream=on)
    dlogits = torch.empty_like(logits)
    M.launch(M.kernels.route_experts_grad, (dlogits, dweights, logits, ids, E, top, 0, 1, 0, 1.0), T, stream=on)
    drouter = normed.float().t() @ dlogits
    by_router = (dlogits @ router.t()).to(H)
    dnormed = combine(dxs, None, row_at, by_router, C, H)
    dx, dscale = torch.empty_like(x), torch.empty(C, device="cuda")
    gargs = (dx, dscale, dnormed, x, scale, None, C, 1, 0, 1e-6)
    M.launch(M.kernels.rms_norm_grad, gargs, T, stream=on,
             workspace=torch.empty(M.workspace_bytes(M.kernels.rms_norm_grad, gargs, T), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    leaf = lambda v: v.double().cpu().requires_grad_()  # noqa: E731
    X, S, Rt, Wt = leaf(x), leaf(scale), leaf(router), leaf(wt)
    n64 = X / torch.sqrt((X * X).mean(1, keepdim=True) + 1e-6) * S
    l64 = n64 @ Rt
    c = ids.cpu().long()
    p = torch.softmax(l64.gather(1, c), 1)
    want = torch.einsum("tj,tjn->tn", p, torch.einsum("tc,tjcn->tjn", n64, Wt[c]))
    want.backward(dy.double().cpu())
    for got, w in ((y, want.detach()), (dx, X.grad), (dscale, S.grad), (drouter, Rt.grad), (dwt, Wt.grad)):
        assert (got.double().cpu() - w).norm() <= 0.03 * w.norm()
