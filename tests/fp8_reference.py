"""Plain 64-bit restatements of the 8-bit quantizer and of the products of its
values, for the tests."""
import torch

TOP = {0: 448.0, 1: 57344.0}
CODE = {0: torch.float8_e4m3fn, 1: torch.float8_e5m2}


def up16(n):
    return -(-n // 16) * 16


def _block_max(x, block):
    """Largest magnitude per block of x (R, C): (R or row blocks, column blocks); NaN wins."""
    r, c = x.shape
    step = 1 if block == 1 else 128
    out = torch.zeros((-(-r // step), -(-c // 128)), dtype=torch.float64)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            out[i, j] = x[i * step:(i + 1) * step, j * 128:(j + 1) * 128].abs().max()
    return out


def quantize(x, block, fmt, pow2):
    """(values of the codes (R, C up to 16), scales) of x (R, C) in the kernel's layout, in float64."""
    x = x.double()
    r, c = x.shape
    a = torch.maximum(_block_max(x, block), torch.tensor(2.0 ** -96, dtype=torch.float64))
    top = TOP[fmt]
    fl = lambda v: v.float().double()  # noqa: E731
    s, inv = fl(a / top), fl(top / a)
    if pow2:
        e = torch.floor(torch.log2(torch.where(torch.isfinite(a), a / top, torch.ones_like(a)))) - 1
        p = torch.exp2(e)
        for _ in range(3):
            p = torch.where(a > top * p, 2 * p, p)
        s, inv = torch.where(torch.isfinite(a), p, s), torch.where(torch.isfinite(a), 1 / p, inv)
    rows = torch.arange(r) // (1 if block == 1 else 128)
    cols = torch.arange(c) // 128
    v = fl(x * inv[rows][:, cols])
    digits, low = ((3, -6), (2, -14))[fmt]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low))) - digits)
    q = torch.zeros((r, up16(c)), dtype=torch.float64)
    q[:, :c] = (torch.round(v / step) * step).clamp(-top, top)
    return q, s.t().contiguous() if block == 1 else s


def values(q, s, block, k):
    """What codes q (R, k up to 16) and scales s stand for, float64."""
    q = q[:, :k].double().cpu()
    s = s.double().cpu()
    blocks = torch.arange(k) // 128
    rows = torch.arange(q.shape[0])
    return q * (s[blocks][:, rows].t() if block == 1 else s[rows // 128][:, blocks])
