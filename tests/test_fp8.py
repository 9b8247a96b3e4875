"""The 8-bit quantizer and the products of its values against 64-bit arithmetic.

Quantizer: the codes and scales are defined to the bit (the roundings to 32 bits of
the scale, its inverse and the scaled value are part of the definition), so they are
compared exactly.

Products: a K block of 128 sums exact products in the tensor core's 32-bit
accumulator. Each of the 128 additions is off by at most one unit of fp32 (2^-23) of
the running sum, whose magnitude the block's sum of |a b| bounds; the scales'
product, the product with it and the addition to the running sum round to nearest
(2^-24 each, the last once per block). With S = sum |a b| over all of K:
|C - exact| <= (128 * 2^-23 + (blocks + 2) * 2^-24) * S, and bf16 adds half a step,
2^-8 of the value.
"""
import numpy as np
import pytest
import torch

import mantle_cuda as M
from fp8_reference import CODE, quantize, up16, values

ptr = lambda n, at=1 << 20: M.DevicePtr(at, n)  # noqa: E731


def q_args(r, c, block=1, both=False, kind=0, fmt=0, pow2=0, rows_of=None, xrows=None, **change):
    rb, cb = -(-r // 128), -(-c // 128)
    n = dict(q=r * up16(c), s=4 * (cb * r if block == 1 else rb * cb), qt=c * up16(r),
             st=4 * (rb * c if block == 1 else rb * cb), x=(xrows or r) * c * (2 if kind else 4))
    n.update(change)
    return [ptr(n["q"]), ptr(n["s"]), ptr(n["qt"]) if both else None, ptr(n["st"]) if both else None, ptr(n["x"]),
            rows_of, r, c, r if xrows is None else xrows, block, kind, fmt, pow2]


@pytest.mark.parametrize("args,nd,match", [
    (q_args(4, 256, block=2), 1, "block must be"),
    (q_args(4, 256, q=4 * 256 - 1), 1, "the codes"),
    (q_args(4, 256, s=4), 1, "the scales"),
    (q_args(4, 256, both=True, qt=256 * 16 - 1), 1, "the transposed codes"),
    (q_args(4, 256, both=True, block=128, st=4), 1, "the transposed scales"),
    (q_args(4, 256, x=100), 1, "the input"),
    (q_args(4, 256), 2, "the codes"),
    (q_args(4, 256, fmt=2), 1, "must be 0 or 1"),
    (q_args(-4, 256), 1, "negative"),
    (q_args(4, 256, xrows=9), 1, "as many rows"),
    (q_args(4, 256, xrows=9, rows_of=ptr(15)), 1, "rows_of"),
    (q_args(4, 256, xrows=9, rows_of=ptr(16)), 2, "batch of one"),
    ([None] + q_args(4, 256)[1:], 1, "codes and the scales"),
    ([None, None] + q_args(4, 256)[2:], 1, "codes and the scales"),
    ([M.DevicePtr((1 << 20) + 8, 1 << 20)] + q_args(4, 256)[1:], 1, "16-byte aligned"),
    # an empty tensor, which has no address, is not an argument left out
    ([ptr(0, 0), ptr(0, 0)] + q_args(4, 256, both=True)[2:], 1, "the codes must be a device buffer"),
    (q_args(4, 256, both=True)[:2] + [ptr(0, 0), ptr(0, 0)] + q_args(4, 256)[4:], 1, "the transposed codes must be"),
    (q_args(4, 256, rows_of=ptr(0, 0)), 1, "rows_of must be a device buffer"),
    (q_args(4, 256, xrows=9, rows_of=ptr(0, 0)), 1, "rows_of must be a device buffer"),
])
def test_quantize_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.quantize_fp8, args, nd)


def g_args(batch, m, n, k, bblock=128, fa=0, fb=0, out=0, **change):
    kb, nb = -(-k // 128), -(-n // 128)
    z = dict(c=batch * m * n * (2 if out == 1 else 4), a=batch * m * up16(k), sa=batch * kb * m * 4, b=batch * n * up16(k),
             sb=batch * kb * 4 * (n if bblock == 1 else nb))
    z.update(change)
    return [ptr(z["c"]), ptr(z["a"]), ptr(z["sa"]), ptr(z["b"]), ptr(z["sb"]), m, n, k, bblock, fa, fb, out]


@pytest.mark.parametrize("args,match", [
    (g_args(1, 4, 5, 129, c=79), "C has"),
    (g_args(1, 4, 5, 129, a=4 * 144 - 1), "A has"),
    (g_args(1, 4, 5, 129, sa=28), "A's scales"),
    (g_args(1, 4, 5, 129, b=5 * 144 - 1), "B has"),
    (g_args(1, 4, 200, 129, sb=12), "B's scales"),
    (g_args(1, 4, 5, 129, bblock=1, sb=36), "B's scales"),
    (g_args(1, 4, 5, 129, bblock=64), "1 or 128 rows"),
    (g_args(1, 4, 5, 129, fa=2), "formats"),
    (g_args(1, 4, 5, 129, out=3), "formats"),
    (g_args(1, 4, -5, 129), "negative"),
])
def test_gemm_fp8_refuses(args, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.gemm_fp8, args, 1)
    with pytest.raises(M.MantleError, match="batch above"):
        M.launch(M.kernels.gemm_fp8, g_args(1, 1, 1, 1, c=0, a=0, sa=0, b=0, sb=0), 70000)


def e_args(groups, t, n, k, out=0, offsets=None, **change):
    g = g_args(1, t, n, k, out=out, b=groups * n * up16(k), sb=groups * -(-k // 128) * -(-n // 128) * 4)
    g[0] = ptr(change.get("y", t * n * (2 if out else 4)))
    return g[:5] + [ptr(4 * (groups + 1) if offsets is None else offsets), t, n, k, 0, 0, out]


@pytest.mark.parametrize("args,groups,match", [
    (e_args(3, 10, 40, 64, y=10), 3, "C has"),
    (e_args(3, 10, 40, 64, offsets=12), 3, "offsets"),
    (e_args(3, 10, 40, 64), 4, "B has"),
    (e_args(2000, 10, 40, 64), 2000, "more than 1024 groups"),
    (e_args(3, 10, 40, 0), 3, "K must be positive"),
])
def test_gemm_grouped_fp8_refuses(args, groups, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.gemm_grouped_fp8, args, groups)


@pytest.mark.parametrize("m,n,k", [(2**31 - 1, 1, 1), (1, 2**31 - 1, 1), (1, 1, 2**31 - 1), (1, 1, 2**31 - 255)])
def test_sizes_that_tiles_would_round_past_32_bits_are_refused(m, n, k):
    # buffers of unknown extent (0 bytes), so that the sizes alone decide
    any_, off = ptr(0), ptr(0)
    with pytest.raises(M.MantleError, match="above 2\\^31 - 256"):
        M.launch(M.kernels.gemm_fp8, [any_] * 5 + [m, n, k, 128, 0, 0, 0], 1)
    with pytest.raises(M.MantleError, match="above 2\\^31 - 256"):
        M.launch(M.kernels.gemm_grouped_fp8, [any_] * 5 + [off, m, n, k, 0, 0, 0], 1)
    for kernel in (M.kernels.gemm_grouped_bf16, M.kernels.gemm_grouped_dx_bf16, M.kernels.gemm_grouped_dw_bf16):
        with pytest.raises(M.MantleError, match="above 2\\^31 - 256"):
            M.launch(kernel, [any_] * 3 + [off, m, n, k, 0], 1)


def test_tensors_are_checked_before_the_call():
    with pytest.raises(M.ArgumentError, match="contiguous CUDA tensor"):
        M.launch(M.kernels.gemm_fp8, [torch.zeros(20)] + g_args(1, 4, 5, 64)[1:], 1)
    with pytest.raises(M.ArgumentError, match="takes 12 arguments"):
        M.launch(M.kernels.gemm_fp8, g_args(1, 4, 5, 64)[:-1], 1)


@pytest.mark.parametrize("nd,match", [(1 << 70, "no ndrange"), ((1, 1, 1, 1), "no ndrange"), ((1, 1), "one-dimensional"), (-1, "negative"), ((), "1-3 dimensions")])
def test_an_ndrange_that_is_none_is_refused(nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.gemm_fp8, g_args(1, 4, 5, 64), nd)


def test_a_launch_takes_buffers_of_the_current_device_only(monkeypatch):
    # a graph's transients have no address of their own; another device's memory may not be reachable
    def made(cls, **fields):
        x = object.__new__(cls)
        vars(x).update(fields)
        return x
    free = made(M.TransientBuffer, dtype=np.dtype(np.uint8), n=64, rid=1)
    for x in (free, M.VirtualBuffer(np.uint8, 64), M.UseHandle(free, 1, 1)):
        with pytest.raises(M.ArgumentError, match="takes a buffer"):
            M.launch(M.kernels.quantize_fp8, [x, ptr(4 * 8)] + q_args(4, 256)[2:], 1)
    M._with_torch()
    monkeypatch.setattr(M, "_current_device", lambda: 0)
    far = made(M.Buffer, dtype=np.dtype(np.uint8), n=1024, ptr=1 << 20, nbytes=1024, dev=made(M.Device, ordinal=1, handle=None), handle=None)
    with pytest.raises(M.ArgumentError, match="argument 1 is a buffer on device 1, the current one is 0"):
        M.launch(M.kernels.quantize_fp8, [far] + q_args(4, 256)[1:], 1)


def test_codes_of_another_format_are_refused(monkeypatch):
    # tensors that say which format their codes are in: the call's format has to be that one
    class Codes:
        def __init__(self, dtype, nbytes=1 << 16):
            self.dtype, self.nbytes = dtype, nbytes
        get_device = lambda self: 0  # noqa: E731
        is_contiguous = lambda self: True  # noqa: E731
        data_ptr = lambda self: 1 << 20  # noqa: E731
    M._with_torch()
    monkeypatch.setattr(M, "_tensor", Codes)
    monkeypatch.setattr(M, "_current_device", lambda: 0)
    e4, e5, u8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8
    quantize_, gemm, grouped = M.kernels.quantize_fp8, M.kernels.gemm_fp8, M.kernels.gemm_grouped_fp8
    name = {0: "e4m3", 1: "e5m2"}
    for fa in (0, 1):
        right, wrong = (e4, e5)[fa], (e5, e4)[fa]
        for kernel, args, at in ((quantize_, q_args(4, 256, both=True, fmt=fa), (0, 2)), (gemm, g_args(1, 4, 5, 64, fa=fa, fb=1 - fa), (1,)),
                                 (gemm, g_args(1, 4, 5, 64, fa=1 - fa, fb=fa), (3,)),
                                 (grouped, e_args(3, 10, 40, 64)[:9] + [fa, 1 - fa, 0], (1,)), (grouped, e_args(3, 10, 40, 64)[:9] + [1 - fa, fa, 0], (3,))):
            for i in at:
                for good in (right, u8):
                    args[i] = Codes(good)
                    assert len(M._operands(kernel, args)) % 4 == 0
                args[i] = Codes(wrong)
                with pytest.raises(M.ArgumentError, match=f"argument {i + 1} holds {wrong}, expected 8-bit codes in {name[fa]}"):
                    M.launch(kernel, args, 1)
                args[i] = ptr(1 << 16)
    for kernel, args, flag in ((gemm, g_args(1, 4, 5, 64), 9), (quantize_, q_args(4, 256), 11)):  # a format that is none: the library's refusal
        args[flag], args[1 if kernel is gemm else 0] = 2, Codes(e5)
        with pytest.raises(M.MantleError, match="formats|must be 0 or 1"):
            M.launch(kernel, args, 1)


# ── on the GPU ───────────────────────────────────────────────────────────────
def stream():
    return torch.cuda.current_stream().cuda_stream


def gpu_quantize(x, block, fmt, pow2, both=False, rows_of=None, only_t=False):
    """Codes (as the format's torch type), scales and their transposed forms of x (batch, R, C) on the GPU."""
    bt, xr, c = x.shape
    r = xr if rows_of is None else rows_of.numel()
    rb, cb = -(-r // 128), -(-c // 128)
    q = torch.full((bt, r, up16(c)), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((bt, cb, r) if block == 1 else (bt, rb, cb), -1.0, device="cuda")
    qt = torch.full((bt, c, up16(r)), 0x55, dtype=torch.uint8, device="cuda")
    st = torch.full((bt, rb, c) if block == 1 else (bt, cb, rb), -1.0, device="cuda")
    outs = ([None, None] if only_t else [q, s]) + ([qt, st] if both or only_t else [None, None])
    M.launch(M.kernels.quantize_fp8, (*outs, x, rows_of, r, c, xr, block, int(x.dtype == torch.bfloat16), fmt, int(pow2)),
             bt, stream=stream())
    torch.cuda.synchronize()
    return q.view(CODE[fmt]), s, qt.view(CODE[fmt]), st


def same(got, want):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, 0.0), torch.nan_to_num(want, 0.0))


def inputs(shape, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale * torch.exp(torch.randn(shape[-1], generator=g))).to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bt,r,c,fmt,pow2", [
    (1, 1, 1, 0, 0), (1, 1, 128, 1, 0), (2, 3, 129, 0, 1), (1, 17, 1000, 1, 1), (1, 128, 128, 0, 0), (3, 130, 257, 0, 0),
    (1, 255, 1028, 1, 0), (1, 5, 15, 0, 1), (1, 2000, 520, 0, 0), (1, 8, 4096, 0, 0), (1, 1300, 1032, 0, 0)])
def test_quantize_matches_the_definition(dev, block, kind, bt, r, c, fmt, pow2):
    x = inputs((bt, r, c), kind, r * 7 + c)
    q, s, qt, st = gpu_quantize(x.cuda(), block, fmt, pow2, both=True)
    q1, s1, _, _ = gpu_quantize(x.cuda(), block, fmt, pow2)
    _, _, qt2, st2 = gpu_quantize(x.cuda(), block, fmt, pow2, only_t=True)
    for b in range(bt):
        wq, ws = quantize(x[b], block, fmt, pow2)
        wt, wst = quantize(x[b].t(), block, fmt, pow2)
        for a, w in ((q[b], wq), (q1[b], wq), (s[b], ws), (s1[b], ws), (qt[b], wt), (qt2[b], wt), (st[b], wst), (st2[b], wst)):
            same(a, w)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("pow2", [0, 1])
@pytest.mark.parametrize("fmt", [0, 1])
def test_quantize_special_values(dev, block, pow2, fmt):
    x = inputs((260, 400), torch.float32, 3)
    x[0, :128] = 0.0                    # a row block of zeros
    x[1, 130] = float("nan")
    x[2, 140] = float("inf")
    x[3, 200] = -float("inf")
    x[4, 256:384] = 1e-42               # subnormal
    x[5, 0] = 3.0e38
    x[6, :128] = 2.0 ** -97             # below the floor
    x[7, :128] = 448.0 * 2.0 ** -20     # a power-of-two scale met exactly
    x[8, 0], x[8, 1:128] = 449.0, 1.0   # just past it
    x[9, :128] = torch.linspace(-1, 1, 128) * 448 / 16  # ties
    x[128:, :] = 0.0                    # whole square blocks of zeros
    q, s, qt, st = gpu_quantize(x[None].cuda(), block, fmt, pow2, both=True)
    wq, ws = quantize(x, block, fmt, pow2)
    wt, wst = quantize(x.t(), block, fmt, pow2)
    for a, w in ((q[0], wq), (s[0], ws), (qt[0], wt), (st[0], wst)):
        same(a, w)
    assert torch.isfinite(s[0][-1, -1] if block == 128 else s[0][0, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("r,c", [(260, 405), (1, 1), (7, 15), (133, 8), (129, 1161), (2000, 523)])
def test_quantize_pads_blocks_of_nan_with_zeros(dev, block, kind, r, c):
    # NaN and infinities in the last block of rows and of columns: what lies between the rows of codes is zeros all the same
    x = inputs((r, c), kind, r + c)
    x[0, c - 1], x[r - 1, 0], x[r - 1, c - 1] = float("nan"), float("nan"), float("nan")
    x[r // 2, c - 1], x[r - 1, c // 2] = float("inf"), float("nan")
    q, s, qt, st = gpu_quantize(x[None].cuda(), block, 0, 0, both=True)
    q1, s1, _, _ = gpu_quantize(x[None].cuda(), block, 0, 0)
    for got, want in ((q, quantize(x, block, 0, 0)[0]), (q1, quantize(x, block, 0, 0)[0]), (qt, quantize(x.t(), block, 0, 0)[0])):
        same(got[0], want)
    for codes, n in ((q, c), (q1, c), (qt, r)):
        assert int(codes.view(torch.uint8)[0, :, n:].max() if up16(n) > n else 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_gathers_rows(dev, block):
    x = inputs((70, 300), torch.bfloat16, 5)
    at = torch.tensor([3, 3, 0, 69, 70, -1, 12, 3] * 20, dtype=torch.int32)  # twice the same, and two that name no row
    q, s, qt, st = gpu_quantize(x[None].cuda(), block, 0, 0, both=True, rows_of=at.cuda())
    named = (at >= 0) & (at < 70)
    full = torch.where(named[:, None], x[at.clamp(0, 69).long()].float(), torch.zeros(()))
    for a, w in zip((q[0], s[0], qt[0], st[0]), quantize(full, block, 0, 0) + quantize(full.t(), block, 0, 0)):
        same(a, w)


@pytest.mark.gpu
def test_quantize_unaligned_input(dev):
    x = inputs((1, 40 * 256 + 1), torch.float32, 6).cuda()
    v = x[0, 1:].view(1, 40, 256)  # starts 4 bytes past an allocation
    assert v.data_ptr() % 16 == 4 and v.is_contiguous()
    q, s, _, _ = gpu_quantize(v, 1, 0, 0)
    wq, ws = quantize(v[0].cpu(), 1, 0, 0)
    same(q[0], wq)
    same(s[0], ws)


def check_product(got, want, total, blocks, out):
    tol = (128 * 2.0 ** -23 + (blocks + 2) * 2.0 ** -24) * total + (2.0 ** -8 * want.abs() if out else 0.0)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - tol).max()
    assert worst <= 0, f"{float(worst):g} past the bound"


def operands(bt, m, n, k, bblock, fa, fb, seed):
    a, b = inputs((bt, m, k), torch.float32, seed), inputs((bt, n, k), torch.float32, seed + 1)
    qa, sa, _, _ = gpu_quantize(a.cuda(), 1, fa, 0)
    qb, sb, _, _ = gpu_quantize(b.cuda(), bblock, fb, 0)
    va = torch.stack([values(qa[i], sa[i], 1, k) for i in range(bt)])
    vb = torch.stack([values(qb[i], sb[i], bblock, k) for i in range(bt)])
    return qa, sa, qb, sb, va, vb


@pytest.mark.gpu
@pytest.mark.parametrize("bblock", [128, 1])
@pytest.mark.parametrize("bt,m,n,k,fa,fb,out", [
    (1, 1, 1, 1, 0, 0, 0), (1, 1, 256, 128, 0, 0, 1), (1, 3, 1000, 520, 1, 0, 0), (2, 16, 384, 1024, 0, 1, 1),
    (1, 17, 129, 257, 0, 0, 0), (3, 200, 264, 72, 0, 0, 0), (1, 128, 256, 640, 1, 1, 1), (1, 300, 515, 1000, 0, 0, 1),
    (2, 1000, 1000, 1000, 0, 0, 0), (1, 129, 4099, 130, 0, 0, 1), (1, 2500, 4200, 384, 0, 0, 0), (1, 5, 4096, 2048, 0, 0, 1),
    (1, 40, 8200, 2056, 0, 0, 0),
    # fewer tiles than SMs: the K blocks split over two to eight CTAs, uneven parts, partial row quarters
    (1, 20, 1000, 4100, 0, 0, 1), (1, 129, 640, 8190, 0, 0, 0), (2, 33, 264, 1100, 1, 0, 1), (1, 256, 8200, 700, 0, 0, 0),
    (1, 65, 77, 2100, 0, 0, 0), (1, 512, 1024, 3000, 0, 0, 1)])
def test_gemm_fp8(dev, bblock, bt, m, n, k, fa, fb, out):
    qa, sa, qb, sb, va, vb = operands(bt, m, n, k, bblock, fa, fb, m + n + k)
    c = torch.full((bt, m, n), float("nan"), dtype=torch.bfloat16 if out else torch.float32, device="cuda")
    M.launch(M.kernels.gemm_fp8, (c, qa, sa, qb, sb, m, n, k, bblock, fa, fb, out), bt, stream=stream())
    torch.cuda.synchronize()
    check_product(c, va @ vb.transpose(1, 2), va.abs() @ vb.abs().transpose(1, 2), -(-k // 128), out)
    assert M.kernel_timeouts() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 600, 3000), (70, 600, 3000), (700, 1500, 900)])
def test_gemm_fp8_gives_the_same_bits_again(dev, m, n, k):
    # split or not, the order of the sums is fixed
    qa, sa, qb, sb, _, _ = operands(1, m, n, k, 128, 0, 0, 5)
    c = torch.full((3, m, n), float("nan"), device="cuda")
    for i in range(3):
        M.launch(M.kernels.gemm_fp8, (c[i], qa, sa, qb, sb, m, n, k, 128, 0, 0, 0), 1, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(c[0], c[1]) and torch.equal(c[0], c[2])


@pytest.mark.gpu
def test_gemm_fp8_empty(dev):
    c = torch.full((2, 3, 8), 5.0, device="cuda")
    z = torch.zeros(256, dtype=torch.uint8, device="cuda")
    s = torch.zeros(64, device="cuda")
    M.launch(M.kernels.gemm_fp8, (c, z, s, z, s, 3, 8, 0, 128, 0, 0, 0), 2, stream=stream())
    torch.cuda.synchronize()
    assert float(c.abs().max()) == 0.0  # the empty sum
    c.fill_(5.0)
    M.launch(M.kernels.gemm_fp8, (c, z, s, z, s, 0, 8, 16, 128, 0, 0, 0), 2, stream=stream())
    M.launch(M.kernels.gemm_fp8, (c, z, s, z, s, 3, 8, 16, 128, 0, 0, 0), 0, stream=stream())
    torch.cuda.synchronize()
    assert float(c.min()) == 5.0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 200])
def test_gemm_fp8_nan_stays_in_its_row_and_column(dev, m):
    qa, sa, qb, sb, va, vb = operands(1, m, 300, 384, 128, 0, 0, 9)
    qa.view(torch.uint8)[0, 1, 200] = 0x7F
    qb.view(torch.uint8)[0, 7, 3] = 0x7F
    c = torch.zeros((1, m, 300), device="cuda")
    M.launch(M.kernels.gemm_fp8, (c, qa, sa, qb, sb, m, 300, 384, 128, 0, 0, 0), 1, stream=stream())
    torch.cuda.synchronize()
    nan = torch.isnan(c[0]).cpu()
    want = torch.zeros((m, 300), dtype=torch.bool)
    want[1], want[:, 7] = True, True
    assert torch.equal(nan, want)


def offsets_of(sizes, first=0):
    o = [first]
    for s in sizes:
        o.append(o[-1] + s)
    return o


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,first,t,n,k,out", [
    ([1], 0, 1, 8, 16, 0),
    ([0, 3, 0, 1], 0, 4, 200, 130, 1),
    ([5, 130, 0, 64, 1], 2, 210, 264, 384, 0),        # rows before the first and behind the last group
    ([128, 256, 127, 129], 0, 640, 515, 1000, 1),
    ([700, 20, 600], 0, 1320, 1024, 256, 0),
    ([2] * 40, 0, 80, 512, 640, 1),
    ([0, 0, 0], 0, 7, 64, 64, 0),
    # many groups of a few rows (rows as the MMA's N operand), some of more than a tile's 32; N past a run of 128 and ragged
    ([1, 0, 33, 5, 0, 2, 70, 16, 1, 1] * 3, 5, 400, 1000, 520, 0),
    ([2] * 60, 0, 120, 515, 1300, 1),
    ([0, 9, 15, 0, 31, 32, 1] * 6, 0, 530, 640, 130, 1),
])
def test_gemm_grouped_fp8(dev, sizes, first, t, n, k, out):
    e = len(sizes)
    x, w = inputs((1, t, k), torch.float32, t), inputs((e, n, k), torch.float32, n)
    qx, sx, _, _ = gpu_quantize(x.cuda(), 1, 0, 0)
    qw, sw, _, _ = gpu_quantize(w.cuda(), 128, 0, 0)
    o = offsets_of(sizes, first)
    y = torch.full((t, n), 3.0, dtype=torch.bfloat16 if out else torch.float32, device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, (y, qx, sx, qw, sw, torch.tensor(o, dtype=torch.int32, device="cuda"), t, n, k, 0, 0, out),
             e, stream=stream())
    torch.cuda.synchronize()
    vx = values(qx[0], sx[0], 1, k)
    got = y.double().cpu()
    for i in range(e):
        lo, hi = o[i], o[i + 1]
        vw = values(qw[i], sw[i], 128, k)
        if hi > lo:
            check_product(got[lo:hi], vx[lo:hi] @ vw.t(), vx[lo:hi].abs() @ vw.abs().t(), -(-k // 128), out)
    assert (got[:o[0]] == 3.0).all() and (got[o[-1]:] == 3.0).all()


@pytest.mark.gpu
def test_gemm_grouped_fp8_bad_offsets_stay_in_bounds(dev):
    # past the end, descending and negative: each clamped to the rows there are
    t, n, k = 100, 136, 256
    x, w = inputs((1, t, k), torch.float32, 1), inputs((4, n, k), torch.float32, 2)
    qx, sx, _, _ = gpu_quantize(x.cuda(), 1, 0, 0)
    qw, sw, _, _ = gpu_quantize(w.cuda(), 128, 0, 0)
    guard = torch.full((t + 64, n), 3.0, device="cuda")
    off = torch.tensor([-5, 40, 20, 90, 1 << 30], dtype=torch.int32, device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, (guard[:t], qx, sx, qw, sw, off, t, n, k, 0, 0, 0), 4, stream=stream())
    torch.cuda.synchronize()
    got, vx = guard.double().cpu(), values(qx[0], sx[0], 1, k)
    assert (got[t:] == 3.0).all()
    for lo, hi, e in ((0, 20, 0), (0, 40, 0), (40, 90, 2), (90, 100, 3)):  # an offset below an earlier one counts as that one
        vw = values(qw[e], sw[e], 128, k)
        check_product(got[lo:hi], vx[lo:hi] @ vw.t(), vx[lo:hi].abs() @ vw.abs().t(), 2, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("fa,fb", [(1, 0), (0, 1), (1, 1)])
@pytest.mark.parametrize("sizes,t,n,k,out", [
    ([130, 0, 64, 1], 200, 264, 384, 1), ([700, 20, 600], 1320, 1024, 250, 0),  # tiles
    ([2] * 60, 120, 515, 1300, 1), ([33, 0, 5, 1] * 20, 790, 640, 130, 0),      # rows as the MMA's N operand
])
def test_gemm_grouped_fp8_in_both_formats(dev, sizes, t, n, k, out, fa, fb):
    # gradients in e5m2 times weight codes in e4m3, and the other pairs
    e, o = len(sizes), offsets_of(sizes)
    qx, sx, _, _ = gpu_quantize(inputs((1, t, k), torch.float32, t).cuda(), 1, fa, 0)
    qw, sw, _, _ = gpu_quantize(inputs((e, n, k), torch.float32, n).cuda(), 128, fb, 0)
    y = torch.full((t, n), 3.0, dtype=torch.bfloat16 if out else torch.float32, device="cuda")
    M.launch(M.kernels.gemm_grouped_fp8, (y, qx, sx, qw, sw, torch.tensor(o, dtype=torch.int32, device="cuda"), t, n, k, fa, fb, out),
             e, stream=stream())
    torch.cuda.synchronize()
    vx, got = values(qx[0], sx[0], 1, k), y.double().cpu()
    for i in range(e):
        r, vw = slice(o[i], o[i + 1]), values(qw[i], sw[i], 128, k)
        if sizes[i]:
            check_product(got[r], vx[r] @ vw.t(), vx[r].abs() @ vw.abs().t(), -(-k // 128), out)
    assert (got[o[-1]:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bblock", [128, 1])
@pytest.mark.parametrize("m,n,k,fa,fb,out", [
    (1, 264, 700, 1, 1, 0), (5, 300, 1300, 1, 1, 1), (9, 136, 2050, 1, 1, 0), (16, 520, 640, 1, 0, 1), (12, 72, 300, 0, 1, 0),  # few rows
    (200, 1000, 3000, 1, 1, 0), (2100, 1100, 300, 1, 1, 1), (40, 500, 2200, 0, 1, 0)])
def test_gemm_fp8_in_both_formats(dev, bblock, m, n, k, fa, fb, out):
    qa, sa, qb, sb, va, vb = operands(1, m, n, k, bblock, fa, fb, m + n)
    c = torch.full((1, m, n), float("nan"), dtype=torch.bfloat16 if out else torch.float32, device="cuda")
    M.launch(M.kernels.gemm_fp8, (c, qa, sa, qb, sb, m, n, k, bblock, fa, fb, out), 1, stream=stream())
    torch.cuda.synchronize()
    check_product(c, va @ vb.transpose(1, 2), va.abs() @ vb.abs().transpose(1, 2), -(-k // 128), out)
