"""The 8-bit and the expert-grouped kernels as they are used together: a graph of two
layers of experts, a linear layer's forward and backward products in 8 bits, graphs,
streams and large buffers."""
import numpy as np
import pytest
import torch

import mantle_cuda as M
from fp8_reference import CODE, quantize, up16, values
from mantle_cuda.workloads import build_experts, route_to_experts, rows_of_codes

U8 = torch.uint8


def test_routes_are_complete_and_in_expert_order():
    rows_of, offsets = route_to_experts(50, 7, 3, 4)
    assert offsets[0] == 0 and offsets[-1] == 150 and (np.diff(offsets) >= 0).all()
    assert sorted(rows_of.tolist()) == sorted(list(range(50)) * 3)
    for e in range(7):  # a token is with an expert once at most
        part = rows_of[offsets[e]:offsets[e + 1]]
        assert len(set(part.tolist())) == len(part)
    assert rows_of_codes(1) == 16 and rows_of_codes(32) == 32


def stream():
    return torch.cuda.current_stream().cuda_stream


def codes(rows, cols, block, bt=1):
    rb, cb = -(-rows // 128), -(-cols // 128)
    return (torch.empty((bt, rows, up16(cols)), dtype=U8, device="cuda"),
            torch.empty((bt, cb, rows) if block == 1 else (bt, rb, cb), device="cuda"))


def quantized(x, block, both=False, rows_of=None, fmt=0):
    bt, xr, c = x.shape
    r = xr if rows_of is None else rows_of.numel()
    q, s = codes(r, c, block, bt)
    qt, st = codes(c, r, block, bt) if both else (None, None)
    M.launch(M.kernels.quantize_fp8, (q, s, qt, st, x, rows_of, r, c, xr, block, int(x.dtype == torch.bfloat16), fmt, 0), bt,
             stream=stream())
    return (q, s, qt, st) if both else (q, s)


def bound(a, b, out):
    """|error| of a @ b summed in K blocks of 128 (see test_fp8.py)."""
    t = (128 * 2.0 ** -23 + (-(-a.shape[1] // 128) + 2) * 2.0 ** -24) * (a.abs() @ b.abs())
    return t + (2.0 ** -8 * (a @ b).abs() if out else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top,width,hidden", [(1, 8, 2, 256, 384), (37, 6, 2, 200, 328), (300, 4, 2, 256, 512)])
def test_two_layers_of_experts(dev, tokens, experts, top, width, hidden):
    w = build_experts(dev, tokens, experts, top, width, hidden, seed=3)
    M.run(w.plan)
    first = w.y.array().copy()
    M.run(w.plan)
    assert np.array_equal(w.y.array(), first)
    # the same launches outside the graph, each stage against 64 bits on what it read
    T, E = tokens * top, experts
    off = torch.from_numpy(w.offsets).cuda()
    wq = {k: quantized(w.tensors[k], 128) for k in ("up", "down")}
    h = torch.zeros((T, hidden), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((T, width), dtype=torch.bfloat16, device="cuda")
    q1, s1 = quantized(w.tensors["x"][None], 1, rows_of=torch.from_numpy(w.rows_of).cuda())
    M.launch(M.kernels.gemm_grouped_fp8, (h, q1, s1, *wq["up"], off, T, hidden, width, 0, 0, 1), E, stream=stream())
    q2, s2 = quantized(h[None], 1)
    M.launch(M.kernels.gemm_grouped_fp8, (y, q2, s2, *wq["down"], off, T, width, hidden, 0, 0, 1), E, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(y.view(torch.int16).cpu().numpy().reshape(-1), first.view(np.int16))
    for q, s, name, out, k in ((q1, s1, "up", h, width), (q2, s2, "down", y, hidden)):
        a = values(q[0].view(CODE[0]), s[0], 1, k)
        for e in range(E):
            r = slice(int(w.offsets[e]), int(w.offsets[e + 1]))
            b = values(wq[name][0][e].view(CODE[0]), wq[name][1][e], 128, k).t()
            assert ((out[r].double().cpu() - a[r] @ b).abs() <= bound(a[r], b, True)).all()
    want, _ = quantize(w.tensors["x"].cpu()[torch.from_numpy(w.rows_of).long()], 1, 0, 0)
    assert torch.equal(q1[0].view(CODE[0]).double().cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,fmt", [(1, 128, 256, 0), (70, 200, 328, 0), (300, 520, 260, 1)])
def test_a_linear_layer_forward_and_backward(dev, m, n, k, fmt):
    g = torch.Generator().manual_seed(m)
    x, wt, dy = (torch.randn(s, generator=g) for s in ((m, k), (n, k), (m, n)))
    xq, xs, xqt, xst = quantized(x[None].cuda(), 1, both=True)
    wq, ws, wqt, wst = quantized(wt[None].cuda(), 128, both=True)
    dq, ds, dqt, dst = quantized(dy[None].cuda().to(torch.bfloat16), 1, both=True, fmt=fmt)
    y, dx, dw = (torch.empty(s, device="cuda") for s in ((m, n), (m, k), (n, k)))
    go = lambda out, a, sa, b, sb, r, c, d, bblock, fa: M.launch(  # noqa: E731
        M.kernels.gemm_fp8, (out, a, sa, b, sb, r, c, d, bblock, fa, 0, 0), 1, stream=stream())
    go(y, xq, xs, wq, ws, m, n, k, 128, 0)
    go(dx, dq, ds, wqt, wst, m, k, n, 128, fmt)
    go(dw, dqt, dst, xqt, xst, n, k, m, 1, fmt)
    torch.cuda.synchronize()
    v = lambda q, s, block, c, f=0: values(q[0].view(CODE[f]), s[0], block, c)  # noqa: E731
    for got, a, b in ((y, v(xq, xs, 1, k), v(wq, ws, 128, k).t()), (dx, v(dq, ds, 1, n, fmt), v(wqt, wst, 128, n).t()),
                      (dw, v(dqt, dst, 1, m, fmt), v(xqt, xst, 1, m).t())):
        assert ((got.double().cpu() - a @ b).abs() <= bound(a, b, False)).all()
    # a square block's transpose is the same values
    assert torch.equal(v(wq, ws, 128, k), v(wqt, wst, 128, n).t())
    # against the gradients of the unquantized layer: a code is off by half a step of its value (2^-4 in e4m3, 2^-3
    # in e5m2) or, below the normal range, of its block's scale (2^-10, 2^-17), so a product of two is off by
    # (1 + r)(1 + q) - 1 of |a| |b| and, for the small ones, less than a further thousandth of the largest products'
    x, wt, dy = x.double(), wt.double(), dy.to(torch.bfloat16).double()
    r = (2.0 ** -4, 2.0 ** -3)[fmt]
    for got, a, b in ((dx, dy, wt), (dw, dy.t(), x)):
        tol = ((1 + r) * (1 + 2.0 ** -4) - 1) * (a.abs() @ b.abs()) + 1e-3 * a.shape[1] * a.abs().max() * b.abs().max()
        assert ((got.double().cpu() - a @ b).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,n,k", [([70, 0, 130, 3], 264, 200), ([3] * 50, 515, 1100)])
def test_an_input_gradient_by_expert_in_8_bits(dev, sizes, n, k):
    # dX = dY W[e]: gradients in e5m2 times the weights' transposed codes, which the quantizer makes with the others
    e, t = len(sizes), sum(sizes)
    o = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    g = torch.Generator().manual_seed(n)
    w, dy = torch.randn((e, n, k), generator=g), torch.randn((1, t, n), generator=g)
    _, _, wqt, wst = quantized(w.cuda(), 128, both=True)
    dq, ds = quantized(dy.cuda().to(torch.bfloat16), 1, fmt=1)
    dx = torch.full((t, k), float("nan"), device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, (dx, dq, ds, wqt, wst, torch.from_numpy(o).cuda(), t, k, n, 1, 0, 0), e, stream=stream())
    torch.cuda.synchronize()
    vd = values(dq[0].view(CODE[1]), ds[0], 1, n)
    for i in range(e):
        r, vw = slice(int(o[i]), int(o[i + 1])), values(wqt[i].view(CODE[0]), wst[i], 128, n).t()
        if sizes[i]:
            assert ((dx[r].double().cpu() - vd[r] @ vw).abs() <= bound(vd[r], vw, False)).all()
            # the codes stand for the weights: off by 2^-4 of a value, or of the block's smallest normal one
            assert ((vw - w[i].double()).abs() <= 2.0 ** -4 * w[i].double().abs() + 2.0 ** -10 * wst[i].max().item()).all()


@pytest.mark.gpu
def test_a_training_step_of_experts_in_a_graph(dev):
    # forward and both gradients as passes of one plan, replayed, against the same launches outside it
    t, e, k, n = 300, 5, 136, 264
    g = torch.Generator(device="cuda").manual_seed(8)
    x, dy, w = (torch.randn(s, generator=g, device="cuda").to(torch.bfloat16) for s in ((t, k), (t, n), (e, k, n)))
    off = np.array([0, 60, 60, 200, 299, 300], np.int32)
    X, DY, W = (M.Buffer.wrap(dev, v, dtype=np.uint16) for v in (x, dy, w))
    O = M.Buffer(dev, off)
    Y, DX, DW = M.Buffer(dev, np.float32, t * n), M.Buffer(dev, np.float32, t * k), M.Buffer(dev, np.uint16, e * k * n)
    graph = M.Graph(dev)
    R, Wr = (lambda p, b: M.use(p, b, read=True)), (lambda p, b: M.use(p, b, write=True))
    M.compute(graph, "forward", lambda p: M.dispatch(p, M.kernels.gemm_grouped_bf16, (Wr(p, Y), R(p, X), R(p, W), R(p, O), t, n, k, 0), e))
    M.compute(graph, "dx", lambda p: M.dispatch(p, M.kernels.gemm_grouped_dx_bf16, (Wr(p, DX), R(p, DY), R(p, W), R(p, O), t, n, k, 0), e))
    M.compute(graph, "dw", lambda p: M.dispatch(p, M.kernels.gemm_grouped_dw_bf16, (Wr(p, DW), R(p, X), R(p, DY), R(p, O), t, n, k, 1), e))
    plan = M.Plan(graph)
    for _ in range(2):
        M.run(plan)
    dev.synchronize()
    o = torch.from_numpy(off).cuda()
    y, dx, dw = torch.empty((t, n), device="cuda"), torch.empty((t, k), device="cuda"), torch.empty((e, k, n), dtype=torch.bfloat16, device="cuda")
    for name, args in (("gemm_grouped_bf16", (y, x, w, o, t, n, k, 0)), ("gemm_grouped_dx_bf16", (dx, dy, w, o, t, n, k, 0)),
                       ("gemm_grouped_dw_bf16", (dw, x, dy, o, t, n, k, 1))):
        M.launch(getattr(M.kernels, name), args, e, stream=stream())
    torch.cuda.synchronize()
    assert np.array_equal(Y.array(), y.cpu().numpy().reshape(-1)) and np.array_equal(DX.array(), dx.cpu().numpy().reshape(-1))
    assert np.array_equal(DW.array().view(np.int16), dw.view(torch.int16).cpu().numpy().reshape(-1))
    with pytest.raises(M.ArgumentError, match="holds float32, expected bfloat16"):
        M.compute(graph, "bad", lambda p: M.dispatch(p, M.kernels.gemm_grouped_bf16, (
            Wr(p, Y), R(p, Y), R(p, W), R(p, O), t, n, k, 0), e))


@pytest.mark.gpu
def test_no_rows_at_all(dev):
    # an empty batch's tensors have no address: every call is a no-op, but a weight gradient is zeros
    e, k, n = 3, 64, 72
    h = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    off, w = torch.zeros(e + 1, dtype=torch.int32, device="cuda"), h(e, k, n)
    M.launch(M.kernels.gemm_grouped_bf16, (h(0, n), h(0, k), w, off, 0, n, k, 1), e, stream=stream())
    M.launch(M.kernels.gemm_grouped_dx_bf16, (h(0, k), h(0, n), w, off, 0, n, k, 1), e, stream=stream())
    dw = torch.full((e, k, n), 5.0, device="cuda")
    M.launch(M.kernels.gemm_grouped_dw_bf16, (dw, h(0, k), h(0, n), off, 0, n, k, 0), e, stream=stream())
    q, s = quantized(torch.zeros((1, 0, k), device="cuda"), 1)
    qw, sw = quantized(torch.zeros((e, n, k), device="cuda"), 128)
    M.launch(M.kernels.gemm_grouped_fp8, (h(0, n), q, s, qw, sw, off, 0, n, k, 0, 0, 1), e, stream=stream())
    M.launch(M.kernels.gemm_fp8, (h(1, 0, n), q, s, qw, sw, 0, n, k, 128, 0, 0, 1), 1, stream=stream())
    torch.cuda.synchronize()
    assert float(dw.abs().max()) == 0.0
    # but not where something would be touched
    with pytest.raises(M.ArgumentError, match="X must be a device buffer"):
        M.launch(M.kernels.gemm_grouped_bf16, (h(4, n), h(0, k), w, off, 4, n, k, 1), e, stream=stream())
    with pytest.raises(M.ArgumentError, match="A must be a device buffer"):
        M.launch(M.kernels.gemm_fp8, (h(1, 4, n), q, s, qw, sw, 4, n, k, 128, 0, 0, 1), 1, stream=stream())


@pytest.mark.gpu
def test_types_strides_and_devices_are_refused(dev):
    e, t, k, n = 2, 16, 64, 72
    x, w = (torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in ((t, k), (e, k, n)))
    y, off = torch.zeros((t, n), device="cuda"), torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    go = lambda *a: M.launch(M.kernels.gemm_grouped_bf16, (*a, t, n, k, 0), e, stream=stream())  # noqa: E731
    go(y, x, w, off)
    go(torch.nn.Parameter(y, requires_grad=False), x, w, off)
    for args, match in (((y, x.half(), w, off), "holds torch.float16, expected bfloat16"), ((y, x, w, off.long()), "expected Int32"),
                        ((y, x, w, off.float()), "expected Int32"), ((y.bfloat16(), x, w, off), "expected Float32"),
                        ((y, x.t().contiguous().t(), w, off), "contiguous"), ((y, x, w.cpu(), off), "current device"),
                        ((y.cpu(), x, w, off), "contiguous CUDA tensor"), ((y, x, w, [0, 1, 2]), "takes a buffer")):
        with pytest.raises(M.ArgumentError, match=match):
            go(*args)
    with pytest.raises(M.ArgumentError, match="no Int32"):
        M.launch(M.kernels.gemm_grouped_bf16, (y, x, w, off, t, n, k, 1 << 40), e, stream=stream())
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_thousand_experts(dev):
    e, k, n = 1024, 64, 72
    sizes = np.arange(e) % 4
    o = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    t = int(o[-1])
    g = torch.Generator().manual_seed(2)
    x, w = torch.randint(-3, 4, (t, k), generator=g).bfloat16(), torch.randint(-3, 4, (e, k, n), generator=g).bfloat16()
    y, off = torch.zeros((t, n), device="cuda"), torch.from_numpy(o).cuda()
    M.launch(M.kernels.gemm_grouped_bf16, (y, x.cuda(), w.cuda(), off, t, n, k, 0), e, stream=stream())
    which = torch.from_numpy(np.repeat(np.arange(e), sizes))
    want = torch.einsum("tk,tkn->tn", x.double(), w[which].double())  # whole numbers: exact
    torch.cuda.synchronize()
    assert torch.equal(y.double().cpu(), want)
    qx, sx = quantized(x[None].cuda().float(), 1)
    qw, sw = quantized(w.transpose(1, 2).contiguous().cuda().float(), 128)
    M.launch(M.kernels.gemm_grouped_fp8, (y, qx, sx, qw, sw, off, t, n, k, 0, 0, 0), e, stream=stream())
    torch.cuda.synchronize()
    vx = values(qx[0].view(CODE[0]), sx[0], 1, k)
    vw = torch.stack([values(qw[i].view(CODE[0]), sw[i], 128, k) for i in range(e)])[which]
    tol = (128 * 2.0 ** -23 + 3 * 2.0 ** -24) * torch.einsum("tk,tnk->tn", vx.abs(), vw.abs())
    assert ((y.double().cpu() - torch.einsum("tk,tnk->tn", vx, vw)).abs() <= tol).all()


@pytest.mark.gpu
def test_captured_and_replayed_on_new_inputs(dev):
    m, n, k = 70, 520, 1300
    xs = [torch.randn((1, m, k), device="cuda") for _ in range(2)]
    wq, ws = quantized(torch.randn((1, n, k), device="cuda"), 128)
    x, c = xs[0].clone(), torch.empty((1, m, n), device="cuda")

    def step(out):
        q, s = codes(m, k, 1)
        M.launch(M.kernels.quantize_fp8, (q, s, None, None, x, None, m, k, m, 1, 0, 0, 0), 1, stream=stream())
        M.launch(M.kernels.gemm_fp8, (out, q, s, wq, ws, m, n, k, 128, 0, 0, 0), 1, stream=stream())

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(c)
    got = []
    for v in xs:
        x.copy_(v)
        graph.replay()
        got.append(c.clone())
    for v, want in zip(xs, got):
        x.copy_(v)
        again = torch.empty_like(c)
        step(again)
        torch.cuda.synchronize()
        assert torch.equal(again, want)
    assert not torch.equal(*got)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(dev):
    t, e, k, n = 600, 8, 512, 768
    x, w = torch.randn((1, t, k), device="cuda"), torch.randn((e, n, k), device="cuda")
    qx, sx = quantized(x, 1)
    qw, sw = quantized(w, 128)
    off = torch.linspace(0, t, e + 1).int().cuda()
    args = lambda out: (out, qx, sx, qw, sw, off, t, n, k, 0, 0, 0)  # noqa: E731
    alone = torch.empty((t, n), device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, args(alone), e, stream=stream())
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros((t, n), device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        M.launch(M.kernels.gemm_grouped_fp8, args(out), e, stream=streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone) for out in outs)


@pytest.mark.gpu
def test_buffers_past_two_to_the_31(dev):
    # 2.2e9 elements: offsets need 64 bits. The last rows and columns against the definition.
    r, c = 540_000, 4096
    x = torch.zeros((1, r, c), dtype=torch.bfloat16, device="cuda")
    x[0, -300:] = torch.randn((300, c), device="cuda").to(torch.bfloat16)
    for block in (1, 128):
        q, s = quantized(x, block)
        torch.cuda.synchronize()
        cut = r - 256 - r % 128  # a multiple of 128
        wq, ws = quantize(x[0, cut:].cpu(), block, 0, 0)
        assert torch.equal(q[0, cut:].view(CODE[0]).double().cpu(), wq)
        assert torch.equal((s[0][:, cut:] if block == 1 else s[0][cut // 128:]).double().cpu(), ws)
        del wq
    # q, s: 128 x 128 blocks. As B of a product: few rows of A, and a tile of them
    for m in (2, 130):
        a = torch.randn((1, m, c), device="cuda")
        qa, sa = quantized(a, 1)
        out = torch.empty((1, m, r), dtype=torch.bfloat16, device="cuda")
        M.launch(M.kernels.gemm_fp8, (out, qa, sa, q, s, m, r, c, 128, 0, 0, 1), 1, stream=stream())
        torch.cuda.synchronize()
        va, vb = values(qa[0].view(CODE[0]), sa[0], 1, c), values(q[0, cut:].view(CODE[0]), s[0][cut // 128:], 128, c).t()
        assert ((out[0, :, cut:].double().cpu() - va @ vb).abs() <= bound(va, vb, True)).all()
        assert float(out[0, :, :cut - 128].abs().max()) == 0.0
        del out
    # as the rows of a grouped product whose last group lies at the end
    w, t = torch.randn((2, 136, c), device="cuda"), r
    del q, s
    qx, sx = quantized(x, 1)
    qw, sw = quantized(w, 128)
    y = torch.full((t, 136), 3.0, device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, (y, qx, sx, qw, sw, torch.tensor([0, 5, t - 7], dtype=torch.int32, device="cuda"), t, 136, c, 0, 0, 0),
             2, stream=stream())
    torch.cuda.synchronize()
    vx, vw = values(qx[0, t - 200:].view(CODE[0]), sx[0][:, t - 200:], 1, c), values(qw[1].view(CODE[0]), sw[1], 128, c).t()
    assert ((y[t - 200:t - 7].double().cpu() - (vx @ vw)[:193]).abs() <= bound(vx, vw, False)[:193]).all()
    assert (y[t - 7:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form,ran_out,m,groups,n,k,out", [
    ("fp8", 1, 512, 0, 1024, 384, 0),              # tiles of 128 rows
    ("fp8", 1, 512, 0, 1024, 384, 1),
    ("fp8", 1, 200, 0, 1024, 4096, 0),             # the K blocks split over a cluster
    ("fp8 grouped", 1, 1100, 3, 1500, 640, 0),
    ("fp8 grouped", 1, 120, 60, 515, 1300, 1),     # rows as the MMA's N operand
    ("fwd", 1, 1100, 3, 2048, 320, 1), ("fwd", 1, 1100, 3, 1096, 1600, 0), ("dx", 1, 1100, 3, 320, 1096, 0), ("dw", 1, 5000, 3, 264, 520, 0),
    ("fwd", 1, 2000, 4, 2560, 320, 1),
    ("fwd", 1, 80, 40, 640, 512, 0), ("dx", 1, 1100, 40, 512, 640, 1),  # rows as the MMA's N operand
    ("fwd", 2, 5120, 2, 776, 520, 1), ("dx", 2, 5120, 2, 1600, 776, 0), ("dw", 2, 4000, 8, 776, 520, 0), ("dw", 2, 9001, 3, 1288, 1032, 1),  # CTA pairs
])
def test_a_wait_that_runs_out_ends_the_launch(dev, form, ran_out, m, groups, n, k, out):
    # The first CTA loads one K block and stops, with the limit of a wait at 20 ms. The launch returns, the CTA (a pair's
    # two) is counted, its tiles (two at most in each case) are not written, or NaN, and every other one has the bits of a
    # launch without the stop; so has the next launch everywhere.
    import time
    g = torch.Generator(device="cuda").manual_seed(m + n)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    dt = torch.bfloat16 if out else torch.float32
    if form == "fp8":
        a, b, c = quantized(rand(1, m, k), 1), quantized(rand(1, n, k), 128), torch.empty((1, m, n), dtype=dt, device="cuda")
        go = lambda: M.launch(M.kernels.gemm_fp8, (c, *a, *b, m, n, k, 128, 0, 0, out), 1, stream=stream())  # noqa: E731
    else:
        off = torch.linspace(0, m, groups + 1).int().cuda()
        if form == "fp8 grouped":
            a, b, c = quantized(rand(1, m, k), 1), quantized(rand(groups, n, k), 128), torch.empty((1, m, n), dtype=dt, device="cuda")
            go = lambda: M.launch(M.kernels.gemm_grouped_fp8, (c, *a, *b, off, m, n, k, 0, 0, out), groups, stream=stream())  # noqa: E731
        else:
            x, dy, w = (v.to(torch.bfloat16) for v in (rand(m, k), rand(m, n), rand(groups, k, n)))
            kernel, a, b, shape = {"fwd": (M.kernels.gemm_grouped_bf16, x, w, (1, m, n)), "dx": (M.kernels.gemm_grouped_dx_bf16, dy, w, (1, m, k)),
                                   "dw": (M.kernels.gemm_grouped_dw_bf16, x, dy, (groups, k, n))}[form]
            c = torch.empty(shape, dtype=dt, device="cuda")
            go = lambda: M.launch(kernel, (c, a, b, off, m, n, k, out), groups, stream=stream())  # noqa: E731
    go()
    torch.cuda.synchronize()
    want = c.clone()
    assert torch.isfinite(want).all()
    c.fill_(float("nan"))
    torch.cuda.synchronize()
    M.kernel_timeouts(reset=True)
    hook = "gemm_fp8" if form.startswith("fp8") else "gemm_grouped_bf16"
    try:
        M.set_wait_limit(20_000_000)
        M.inject_stall(hook, 1)
        t0 = time.perf_counter()
        go()
        torch.cuda.synchronize()
        took = time.perf_counter() - t0
    finally:
        M.inject_stall(hook, 0)
        M.set_wait_limit(0)
    assert M.kernel_timeouts(reset=True) == ran_out
    assert took < 1.0
    lost = torch.isnan(c)
    assert bool(lost[0, 0, 0]) and int(lost.sum()) <= 2 * 256 * 256 and int(lost.sum()) < lost.numel()
    assert torch.equal(c[~lost], want[~lost])
    c.fill_(float("nan"))
    go()
    torch.cuda.synchronize()
    assert torch.equal(c, want) and M.kernel_timeouts() == 0
