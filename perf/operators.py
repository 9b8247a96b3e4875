"""The 8-bit and the expert-grouped matrix products, as cases to be timed.

Four operators, each in its plain form (elementary torch operations in 32 bits) and as calls of this
framework's kernels:

* quantize    `quantize_fp8`: values in blocks of 128 brought to 8-bit floating point with one scale a block.
              A block is 1 x 128 along a row (`block` 1) or 128 x 128 (`block` 128). With a the block's largest
              magnitude (at least 2^-96) and L the format's largest value (448 for e4m3, 57344 for e5m2):
              scale = fl32(a / L), code = round(fl32(x * fl32(L / a))), ties to even. `pow2`: the scale is the
              smallest power of two with a <= L * scale, and code = round(x / scale). `both`: the transposed
              values too, in blocks along the columns. `gather`: row r is row rows[r] of the input.
* gemm_fp8    C = A . B^T of such values, in 32-bit sums; B's scales are 128 x 128 (`bblock` 128) or 1 x 128.
* grouped     `gemm_grouped_bf16` and its gradients: rows offsets[e] .. offsets[e+1] of X times W[e].
* grouped_fp8 `gemm_grouped_fp8`: the same product of 8-bit rows with 8-bit weights W[e] (N x K).
"""
import math
import os
import random
import sys

import torch

own = False

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FORMAT = {"e4m3": 0, "e5m2": 1}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TYPE = {"f32": 0, "bf16": 1}
SMALLEST = 2.0 ** -96


# ── the cases ────────────────────────────────────────────────────────────────
def listed():
    return [
        # the activations of a batch of 32 sequences, one token each, ahead of an 8-bit product
        _q("quantize, 32 tokens", 32, 4096, "bf16", 1, "e4m3", False, False),
        # a training step's activations: row blocks for the forward product, column blocks for the weight gradient
        _q("quantize, 8192 rows both ways", 8192, 4096, "bf16", 1, "e4m3", False, True),
        # weights held in 32 bits, in square blocks with power-of-two scales, and their transpose; odd sizes
        _q("quantize, weights 5001 x 4100", 5001, 4100, "f32", 128, "e4m3", True, True),
        # one token through a linear layer: the weights are read once
        _g("fp8, one token", 1, 1, 8192, 4096, 128, "e4m3", "e4m3", "bf16"),
        # the benchmark's GEMM size
        _g("fp8, 8192 cubed", 1, 8192, 8192, 8192, 128, "e4m3", "e4m3", "bf16"),
        # two weight gradients over an odd number of tokens: both sides in row blocks, gradients in e5m2, 32-bit sums out
        _g("fp8, weight gradients", 2, 2047, 4100, 5001, 1, "e5m2", "e4m3", "f32"),
        # a step of 64 sequences over 32 experts: two rows an expert, the experts' weights are what is read
        _r("experts bf16, 64 tokens", "fwd", 64, 32, 2048, 4096, "bf16"),
        # a training batch over 16 experts of ragged sizes, one of them empty: forward and both gradients
        _r("experts bf16, forward", "fwd", 8192, 16, 2048, 4096, "bf16"),
        _r("experts bf16, input gradient", "dx", 8192, 16, 2048, 4096, "bf16"),
        _r("experts bf16, weight gradient", "dw", 8191, 16, 2048, 4096, "f32"),
        # the same step and a prompt's rows with the experts held in 8 bits
        _e("experts fp8, 128 tokens", 128, 64, 4096, 2048, "bf16"),
        _e("experts fp8, 8191 rows", 8191, 16, 4096, 4096, "bf16"),
    ]


def _q(name, rows, cols, kind, block, fmt, pow2, both, gather=False):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "type": kind, "block": block, "fmt": fmt, "pow2": pow2, "both": both, "gather": gather}


def _g(name, batch, m, n, k, bblock, fa, fb, out):
    return {"name": name, "op": "gemm_fp8", "batch": batch, "m": m, "n": n, "k": k, "bblock": bblock, "fa": fa, "fb": fb, "out": out}


def _r(name, way, t, experts, k, n, out):
    return {"name": name, "op": "grouped", "way": way, "t": t, "experts": experts, "k": k, "n": n, "out": out}


def _e(name, t, experts, k, n, out):
    return {"name": name, "op": "grouped_fp8", "t": t, "experts": experts, "k": k, "n": n, "out": out}


def draw(rng):
    def size(lo, hi, step=1):  # over the logarithm
        return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)

    op = rng.choice(("quantize", "gemm_fp8", "grouped", "grouped_fp8"))
    if op == "quantize":
        c = _q("", size(1, 8192), size(128, 8192), rng.choice(("bf16", "f32")), rng.choice((1, 128)), rng.choice(("e4m3", "e5m2")),
               rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.25)
    elif op == "gemm_fp8":
        bblock = rng.choice((1, 128))
        c = _g("", rng.choice((1, 1, 2)), size(1, 4096), size(128, 8192), size(128, 8192), bblock, rng.choice(("e4m3", "e5m2")),
               "e4m3", rng.choice(("bf16", "bf16", "f32")))
    elif op == "grouped":
        c = _r("", rng.choice(("fwd", "dx", "dw")), size(8, 8192), size(4, 32), size(256, 2048, 8), size(256, 4096, 8), rng.choice(("bf16", "bf16", "f32")))
    else:
        c = _e("", size(8, 8192), size(4, 64), size(256, 4096), size(256, 4096), "bf16")
    del c["name"]
    return c


# ── inputs ───────────────────────────────────────────────────────────────────
def _up(n, to):
    return -(-n // to) * to


def _sizes(t, experts, seed):
    """Rows of each expert: uneven by up to a factor of three, one expert empty; their sum is t."""
    rng = random.Random(seed)
    share = [rng.uniform(0.5, 1.5) for _ in range(experts)]
    share[rng.randrange(experts)] = 0.0
    total, at, sizes = sum(share), 0.0, []
    for s in share:
        sizes.append(round(t * (at + s) / total) - round(t * at / total))
        at += s
    return sizes


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    op = case["op"]
    s = dict(case)
    if op == "quantize":
        r, c, b = case["rows"], case["cols"], case["block"]
        x = normal(r, c) * (1.0 + 20.0 * (torch.rand(c, generator=g, device="cuda") < 0.004))  # a few wide channels
        s["x"] = x.to(TYPES[case["type"]])
        s["rows_of"] = torch.randint(0, r, (r,), generator=g, device="cuda", dtype=torch.int32) if case["gather"] else None
        rb, cb, code = -(-r // 128), -(-c // 128), CODES[case["fmt"]]
        s["q"] = torch.empty((r, _up(c, 16)), dtype=torch.uint8, device="cuda").view(code)
        s["s"] = torch.empty((cb, r) if b == 1 else (rb, cb), device="cuda")
        if case["both"]:
            s["qt"] = torch.empty((c, _up(r, 16)), dtype=torch.uint8, device="cuda").view(code)
            s["st"] = torch.empty((rb, c) if b == 1 else (cb, rb), device="cuda")
    elif op == "gemm_fp8":
        bt, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        s["a"], s["sa"] = _codes(normal(bt, m, k), 1, case["fa"])
        s["b"], s["sb"] = _codes(normal(bt, n, k), case["bblock"], case["fb"])
        s["c"] = torch.empty((bt, m, n), dtype=TYPES[case["out"]], device="cuda")
    else:
        t, e, k, n = case["t"], case["experts"], case["k"], case["n"]
        sizes = _sizes(t, e, seed)
        s["cap"] = max(sizes)
        s["offsets"] = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
        if op == "grouped":
            way, out = case["way"], TYPES[case["out"]]
            if way != "dx":
                s["x"] = normal(t, k).to(torch.bfloat16)
            if way != "fwd":
                s["dy"] = normal(t, n).to(torch.bfloat16)
            if way != "dw":
                s["w"] = (normal(e, k, n) / math.sqrt(k)).to(torch.bfloat16)
            s["y"] = torch.empty({"fwd": (t, n), "dx": (t, k), "dw": (e, k, n)}[way], dtype=out, device="cuda")
        else:
            s["a"], s["sa"] = _codes(normal(t, k), 1, "e4m3")
            s["b"], s["sb"] = _codes(normal(e, n, k) / math.sqrt(k), 128, "e4m3")
            s["y"] = torch.empty((t, n), dtype=TYPES[case["out"]], device="cuda")
    return s


def _codes(x, block, fmt):
    """8-bit codes (rows a multiple of 16 bytes apart) and scales of x (..., rows, cols)."""
    lead = x.shape[:-2]
    x = x.reshape(-1, *x.shape[-2:])
    q, s = _quantize(x, block, fmt, False)
    return q.view(*lead, *q.shape[1:]), s.view(*lead, *s.shape[1:])


# ── the plain forms ──────────────────────────────────────────────────────────
def _quantize(x, block, fmt, pow2):
    """Codes (b, rows, cols up to 16) and scales of x (b, rows, cols): (b, col blocks, rows) for row blocks, (b, row blocks, col blocks) for square ones."""
    b, r, c = x.shape
    br, rp, cp = (1, r, _up(c, 128)) if block == 1 else (128, _up(r, 128), _up(c, 128))
    x = torch.nn.functional.pad(x.float(), (0, cp - c, 0, rp - r)).view(b, rp // br, br, cp // 128, 128)
    a = x.abs().amax(dim=(2, 4)).clamp(min=SMALLEST)
    top = LARGEST[fmt]
    if pow2:
        mant, exp = torch.frexp(a)
        exp = exp - (9 if fmt == "e4m3" else 16) + (mant > 0.875)
        scale, inv = torch.ldexp(torch.ones_like(a), exp), torch.ldexp(torch.ones_like(a), -exp)
    else:
        top = torch.full_like(a, top)  # a tensor: a quotient with a number is a product with its rounded inverse
        scale, inv = a / top, top / a
    q = (x * inv[:, :, None, :, None]).view(b, rp, cp)[:, :r, :c]
    q = torch.nn.functional.pad(q, (0, _up(c, 16) - c)).to(CODES[fmt])
    return q, (scale.transpose(1, 2) if block == 1 else scale).contiguous()


def _values(q, s, block, k):
    """The 32-bit values that codes q (b, rows, k up to 16) and scales s stand for."""
    q = q[..., :k].float()
    s = s.transpose(-1, -2) if block == 1 else s.repeat_interleave(128, -2)[:, : q.shape[-2]]
    return q * s.repeat_interleave(128, -1)[..., :k]


def _spread(x, offsets, cap):
    """Rows (t, c) of each group in a block of its own, (groups, cap, c) in 32 bits, zeros below them; and where each row came from."""
    at = offsets[:-1, None].long() + torch.arange(cap, device=x.device)
    inside = at < offsets[1:, None]
    rows = torch.where(inside, at, x.shape[0])
    return torch.cat((x.float(), x.new_zeros((1, x.shape[1]), dtype=torch.float32)))[rows], rows


def _gather(blocks, rows, t):
    """The rows of _spread's blocks back in their places."""
    y = blocks.new_empty((t + 1, blocks.shape[-1]))
    y[rows.reshape(-1)] = blocks.reshape(-1, blocks.shape[-1])
    return y[:t]


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "quantize":
        x = state["x"] if state["rows_of"] is None else state["x"][state["rows_of"].long()]
        q, s = _quantize(x[None], state["block"], state["fmt"], state["pow2"])
        if not state["both"]:
            return {"q": q[0], "s": s[0]}
        qt, st = _quantize(x.t()[None], state["block"], state["fmt"], state["pow2"])
        return {"q": q[0], "s": s[0], "qt": qt[0], "st": st[0]}
    if op == "gemm_fp8":
        a = _values(state["a"], state["sa"], 1, state["k"])
        b = _values(state["b"], state["sb"], state["bblock"], state["k"])
        return torch.matmul(a, b.transpose(1, 2)).to(TYPES[state["out"]])
    out, t, offsets, cap = TYPES[state["out"]], state["t"], state["offsets"], state["cap"]
    if op == "grouped_fp8":
        x, rows = _spread(_values(state["a"][None], state["sa"][None], 1, state["k"])[0], offsets, cap)
        w = _values(state["b"], state["sb"], 128, state["k"])
        return _gather(torch.bmm(x, w.transpose(1, 2)), rows, t).to(out)
    if state["way"] == "fwd":
        x, rows = _spread(state["x"], offsets, cap)
        return _gather(torch.bmm(x, state["w"].float()), rows, t).to(out)
    dy, rows = _spread(state["dy"], offsets, cap)
    if state["way"] == "dx":
        return _gather(torch.bmm(dy, state["w"].float().transpose(1, 2)), rows, t).to(out)
    x, _ = _spread(state["x"], offsets, cap)
    return torch.bmm(x.transpose(1, 2), dy).to(out)


# ── this framework's kernels ─────────────────────────────────────────────────
def _own(state):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mantle.jl_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mantle_cuda as M

    stream, op, k = torch.cuda.current_stream().cuda_stream, state["op"], M.kernels
    if op == "quantize":
        both = state["both"]
        M.launch(k.quantize_fp8, (state["q"], state["s"], state["qt"] if both else None, state["st"] if both else None, state["x"], state["rows_of"],
                                  state["rows"], state["cols"], state["rows"], state["block"], TYPE[state["type"]], FORMAT[state["fmt"]],
                                  int(state["pow2"])), 1, stream=stream)
        return {"q": state["q"], "s": state["s"], "qt": state["qt"], "st": state["st"]} if both else {"q": state["q"], "s": state["s"]}
    if op == "gemm_fp8":
        M.launch(k.gemm_fp8, (state["c"], state["a"], state["sa"], state["b"], state["sb"], state["m"], state["n"], state["k"], state["bblock"],
                              FORMAT[state["fa"]], FORMAT[state["fb"]], TYPE[state["out"]]), state["batch"], stream=stream)
        return state["c"]
    sizes = (state["offsets"], state["t"], state["n"], state["k"])
    if op == "grouped_fp8":
        M.launch(k.gemm_grouped_fp8, (state["y"], state["a"], state["sa"], state["b"], state["sb"], *sizes, 0, 0, TYPE[state["out"]]),
                 state["experts"], stream=stream)
        return state["y"]
    kernel, one, two = {"fwd": (k.gemm_grouped_bf16, "x", "w"), "dx": (k.gemm_grouped_dx_bf16, "dy", "w"),
                        "dw": (k.gemm_grouped_dw_bf16, "x", "dy")}[state["way"]]
    M.launch(kernel, (state["y"], state[one], state[two], *sizes, TYPE[state["out"]]), state["experts"], stream=stream)
    return state["y"]


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    op = case["op"]
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        rb, cb = -(-r // 128), -(-c // 128)
        per = {"bf16": 2, "f32": 4}[case["type"]]
        out = r * _up(c, 16) + 4 * (cb * r if case["block"] == 1 else rb * cb)
        if case["both"]:
            out += c * _up(r, 16) + 4 * (rb * c if case["block"] == 1 else rb * cb)
        return {"bytes": r * c * per + out + (4 * r if case["gather"] else 0), "flops": 3 * r * c}
    wide = {"bf16": 2, "f32": 4}[case["out"]]
    if op == "gemm_fp8":
        b, m, n, k = case["batch"], case["m"], case["n"], case["k"]
        kb, nb = -(-k // 128), -(-n // 128)
        scales = kb * m + kb * (n if case["bblock"] == 1 else nb)
        return {"bytes": b * (m * k + n * k + 4 * scales + m * n * wide), "flops": 2 * b * m * n * k}
    t, e, k, n = case["t"], case["experts"], case["k"], case["n"]
    used = min(e - 1, t)  # one expert has no rows
    if op == "grouped_fp8":
        kb, nb = -(-k // 128), -(-n // 128)
        return {"bytes": t * k + 4 * kb * t + used * (n * k + 4 * kb * nb) + t * n * wide, "flops": 2 * t * n * k}
    if case["way"] == "dw":
        return {"bytes": 2 * t * (k + n) + e * k * n * wide, "flops": 2 * t * n * k}
    rows_in, rows_out = (k, n) if case["way"] == "fwd" else (n, k)
    return {"bytes": 2 * t * rows_in + 2 * used * k * n + t * rows_out * wide, "flops": 2 * t * n * k}


# ── in 64 bits ───────────────────────────────────────────────────────────────
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double()
        if case["gather"]:
            x = x.index_select(0, s["rows_of"].long())
        way = (case["block"], case["fmt"], case["pow2"])
        q, sc = _exact_codes(x, *way)
        if not case["both"]:
            return {"q": q, "s": sc}
        qt, st = _exact_codes(x.t().contiguous(), *way)
        return {"q": q, "s": sc, "qt": qt, "st": st}
    if op == "gemm_fp8":
        return torch.stack([_exact_values(s["a"][i], s["sa"][i], 1, case["k"]) @ _exact_values(s["b"][i], s["sb"][i], case["bblock"], case["k"]).t()
                            for i in range(case["batch"])])
    at = s["offsets"].tolist()
    parts = []
    for e in range(case["experts"]):
        lo, hi = at[e], at[e + 1]
        if op == "grouped_fp8":
            x = _exact_values(s["a"][lo:hi], s["sa"][:, lo:hi], 1, case["k"])
            parts.append(x @ _exact_values(s["b"][e], s["sb"][e], 128, case["k"]).t())
        elif case["way"] == "fwd":
            parts.append(s["x"][lo:hi].double() @ s["w"][e].double())
        elif case["way"] == "dx":
            parts.append(s["dy"][lo:hi].double() @ s["w"][e].double().t())
        else:
            parts.append(s["x"][lo:hi].double().t() @ s["dy"][lo:hi].double())
    return torch.stack(parts) if case.get("way") == "dw" else torch.cat(parts)


def _exact_values(q, s, block, k):
    rows = torch.arange(q.shape[0], device=q.device)
    blocks = torch.arange(k, device=q.device) // 128
    s = s.double()
    scale = s[blocks][:, rows].t() if block == 1 else s[rows // 128][:, blocks]
    return q[:, :k].double() * scale


def _exact_codes(x, block, fmt, pow2):
    """The codes' values and the scales of x (rows, cols) in 64 bits. The operator's own roundings to 32 bits
    (the scale, its inverse, the scaled value) are part of its definition and are made here too."""
    r, c = x.shape
    fl32 = lambda v: v.float().double()  # noqa: E731
    col = torch.arange(c, device=x.device) // 128
    cb = int(col[-1]) + 1
    a = torch.zeros((r, cb), dtype=torch.float64, device=x.device)
    a.scatter_reduce_(1, col.expand(r, c), x.abs(), "amax")
    row = torch.arange(r, device=x.device) // (1 if block == 1 else 128)
    if block != 1:
        wide = torch.zeros((int(row[-1]) + 1, cb), dtype=torch.float64, device=x.device)
        a = wide.scatter_reduce_(0, row[:, None].expand(r, cb), a, "amax")
    a = torch.maximum(a, torch.full_like(a, SMALLEST))
    top = LARGEST[fmt]
    if pow2:
        scale = torch.exp2(torch.floor(torch.log2(a / top)) - 1)
        for _ in range(3):
            scale = torch.where(a > top * scale, 2 * scale, scale)
        inv = 1 / scale
    else:
        scale, inv = fl32(a / top), fl32(top / a)
    v = fl32(x * inv[row][:, col])
    digits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low))) - digits)
    q = torch.zeros((r, _up(c, 16)), dtype=torch.float64, device=x.device)
    q[:, :c] = (torch.round(v / step) * step).clamp(-top, top)
    return q, scale.t().contiguous() if block == 1 else scale
