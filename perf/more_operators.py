"""What surrounds the products by expert, as cases to be timed.

Six calls of three operators, each in its plain form (elementary torch operations in 32 bits, the choice of
experts in 64) and as calls of this framework's kernels:

* norm      `rms_norm`: h = x + residual, y = h * rsqrt(mean(h^2) + eps) * w by row, y from the 32-bit h. Outputs: h
            and y in x's type, and y in 8 bits with a scale for each 1 x 128 block, as `quantize_fp8` makes them.
* norm_grad `rms_norm_grad`: dx and dw of y = h * rsqrt(mean(h^2) + eps) * w, with the gradient that reaches h by
            the residual path added to dx.
* route     `route_experts`: from logits the experts of each token and their weights, and the rows' order by
            expert. Scores are softmax or sigmoid of the logits; a bias is added for the choice alone; of `groups`
            groups the `top_groups` with the largest sums of their `best` best keys stay; the `top` largest keys
            are chosen, ties to the lower index; weights are the chosen scores, over their sum where `renorm`, times
            `scale`. A token that is not live takes no expert: -1, weights 0. The rows are the chosen slots in the
            order of expert, then token: offsets by expert, the token of each row, the row of each slot.
* route_grad `route_experts_grad`: the logits' gradient from the weights'.
* combine   `combine_experts`: y[t] = base[t] + sum over j of w[t, j] * rows[row_at[t, j]].
* combine_grad `combine_experts_grad`: the gradients of the rows and of the weights.
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
SCORE = {"softmax": 0, "sigmoid": 1}
SMALLEST = 2.0 ** -96
EPS = 1e-6


# ── the cases ────────────────────────────────────────────────────────────────
def listed():
    return [
        # a decode step of 32 sequences: the residual's addition and the 8-bit operand of the next product
        _n("norm, 32 tokens to 8 bits", 32, 4096, "bf16", "bf16", True, False, "e4m3"),
        # a training step's tokens: the residual, y for the router and the backward pass, codes for the products
        _n("norm, 8192 rows, residual", 8192, 4096, "bf16", "bf16", True, True, "e4m3"),
        # a last norm in 32 bits, odd sizes
        _n("norm, 5001 x 4013 in 32 bits", 5001, 4013, "f32", "f32", False, True, ""),
        # that training step backward: the residual path's gradient is added
        _m("norm gradient, 8192 rows", 8192, 4096, "bf16", "bf16", True),
        _m("norm gradient, 1023 x 5001", 1023, 5001, "f32", "f32", False),
        # a decode step of 64 sequences over 32 experts
        _r("route, 64 tokens", 64, 32, 2, 1, 1, 1, "softmax", True, False, False, "f32"),
        # a training step over many experts in groups, balanced by a bias; the last tokens of the batch are padding
        _r("route, 8192 tokens, groups", 8192, 256, 8, 8, 4, 2, "sigmoid", True, True, True, "f32"),
        # a ragged batch's logits backward, scores over all experts
        _s("route gradient, 8191 tokens", 8191, 64, 6, "softmax", False, "bf16"),
        # the decode step's rows back to their tokens
        _c("combine, 64 tokens", 64, 2048, 2, "bf16", "bf16", True, True),
        # a training step: rows back to their tokens, with the residual; and its backward
        _c("combine, 8192 tokens", 8192, 2048, 8, "bf16", "bf16", True, True),
        _d("combine gradient, 8192 tokens", 8192, 2048, 8, "bf16", "bf16"),
        _d("combine gradient, 1021 x 4104", 1021, 4104, 2, "f32", "f32"),
    ]


def _n(name, rows, cols, kind, wkind, residual, y, fmt):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "type": kind, "wtype": wkind, "residual": residual, "y": y, "fmt": fmt}


def _m(name, rows, cols, kind, wkind, residual):
    return {"name": name, "op": "norm_grad", "rows": rows, "cols": cols, "type": kind, "wtype": wkind, "residual": residual}


def _r(name, t, experts, top, groups, top_groups, best, score, renorm, bias, padded, kind):
    return {"name": name, "op": "route", "t": t, "experts": experts, "top": top, "groups": groups, "top_groups": top_groups, "best": best,
            "score": score, "renorm": renorm, "bias": bias, "padded": padded, "type": kind}


def _s(name, t, experts, top, score, renorm, kind):
    return {"name": name, "op": "route_grad", "t": t, "experts": experts, "top": top, "score": score, "renorm": renorm, "type": kind}


def _c(name, t, cols, top, kind, ykind, base, weighted):
    return {"name": name, "op": "combine", "t": t, "cols": cols, "top": top, "type": kind, "ytype": ykind, "base": base, "weighted": weighted}


def _d(name, t, cols, top, kind, ykind):
    return {"name": name, "op": "combine_grad", "t": t, "cols": cols, "top": top, "type": kind, "ytype": ykind}


def draw(rng):
    def size(lo, hi):  # over the logarithm
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind, flip = (lambda: rng.choice(("bf16", "f32"))), (lambda: rng.random() < 0.5)
    op = rng.choice(("norm", "norm_grad", "route", "route_grad", "combine", "combine_grad"))
    if op == "norm":
        fmt = rng.choice(("", "e4m3", "e5m2"))
        c = _n("", size(1, 8192), size(64, 8192), kind(), kind(), flip(), fmt == "" or flip(), fmt)
    elif op == "norm_grad":
        c = _m("", size(1, 8192), size(64, 8192), kind(), kind(), flip())
    elif op == "route":
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * size(-(-8 // groups), 256 // groups)
        top = rng.randint(1, 8)
        need = -(-top * groups // experts)  # groups that hold enough experts
        c = _r("", size(1, 8192), experts, top, groups, rng.randint(need, groups), rng.randint(1, min(2, experts // groups)),
               rng.choice(("softmax", "sigmoid")), flip(), flip(), flip(), kind())
    elif op == "route_grad":
        c = _s("", size(1, 8192), size(8, 256), rng.randint(1, 8), rng.choice(("softmax", "sigmoid")), flip(), kind())
    elif op == "combine":
        c = _c("", size(1, 8192), size(64, 4096), rng.randint(1, 8), kind(), kind(), flip(), flip())
    else:
        c = _d("", size(1, 8192), size(64, 4096), rng.randint(1, 8), kind(), kind())
    del c["name"]
    length = "rows" if "rows" in c else "t"
    c[length] = min(c[length], 1024 * 500_000_000 // work({**c, length: 1024})["bytes"])  # half a gigabyte at most
    return c


# ── inputs ───────────────────────────────────────────────────────────────────
def _up(n, to):
    return -(-n // to) * to


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    op, s = case["op"], dict(case)
    kind = TYPES[case["type"]]
    if op in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        x = normal(r, c) * (1.0 + 20.0 * (torch.rand(c, generator=g, device="cuda") < 0.004))  # a few wide channels
        s["w"] = (1.0 + 0.1 * normal(c)).to(TYPES[case["wtype"]])
        if op == "norm":
            s["x"], s["res"] = x.to(kind), (2.0 * normal(r, c)).to(kind) if case["residual"] else None
            s["y"] = empty(r, c, dtype=kind) if case["y"] else None
            s["h"] = empty(r, c, dtype=kind) if case["residual"] else None
            fmt = case["fmt"]
            s["q"] = empty(r, _up(c, 16), dtype=torch.uint8).view(CODES[fmt]) if fmt else None
            s["s"] = empty(-(-c // 128), r) if fmt else None
        else:
            s["h"], s["dy"] = x.to(kind), normal(r, c).to(kind)
            s["dres"] = normal(r, c).to(kind) if case["residual"] else None
            s["dx"], s["dw"] = empty(r, c, dtype=kind), empty(c)
        return s
    t, k = case["t"], case["top"]
    if op in ("route", "route_grad"):
        e = case["experts"]
        s["logits"] = (1.5 * normal(t, e) + 0.5 * normal(e)).to(kind)  # some experts are liked more than others
        s["ids"], s["weights"] = empty(t, k, dtype=torch.int32), empty(t, k)
        if op == "route":
            s["bias_of"] = 0.05 * normal(e) if case["bias"] else None
            s["live"] = (torch.arange(t, device="cuda") < t - seed % (1 + t // 8)).to(torch.int32) if case["padded"] else None
            s["scale"] = 2.5 if case["renorm"] and case["score"] == "sigmoid" else 1.0
            s["offsets"], s["rows_of"], s["row_at"] = (empty(n, dtype=torch.int32) for n in (e + 1, t * k, t * k))
        else:
            s["scale"] = 1.0
            s["ids"] = s["logits"].float().argsort(1, descending=True)[:, :k].to(torch.int32).contiguous()
            s["dweights"], s["dlogits"] = normal(t, k), empty(t, e, dtype=kind)
        return s
    c, e, ykind = case["cols"], 32, TYPES[case["ytype"]]
    ids = torch.rand((t, e), generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32)
    _, s["rows_of"], s["row_at"] = _order(ids, e)
    w = torch.rand((t, k), generator=g, device="cuda") + 0.05
    s["w"] = w / w.sum(1, keepdim=True) if case.get("weighted", True) else None
    s["rows"] = normal(t * k, c).to(kind)
    if op == "combine":
        s["base_of"] = normal(t, c).to(ykind) if case["base"] else None
        s["out"] = empty(t, c, dtype=ykind)
    else:
        s["dy"] = normal(t, c).to(ykind)
        s["drows"], s["dweights"] = empty(t * k, c, dtype=kind), empty(t, k)
    return s


# ── the plain forms ──────────────────────────────────────────────────────────
def _quantize(y, fmt):
    """Codes (rows, cols up to 16) and scales (blocks, rows) of y (rows, cols) in 32 bits, one scale for each 1 x 128 block."""
    r, c = y.shape
    cp = _up(c, 128)
    y = torch.nn.functional.pad(y, (0, cp - c)).view(r, cp // 128, 128)
    a = y.abs().amax(dim=2).clamp(min=SMALLEST)
    top = torch.full_like(a, LARGEST[fmt])  # a tensor: a quotient with a number is a product with its rounded inverse
    q = (y * (top / a)[:, :, None]).view(r, cp)[:, :c]
    q = torch.nn.functional.pad(q, (0, _up(c, 16) - c)).to(CODES[fmt])
    return q, (a / top).t().contiguous()


def _order(ids, experts):
    """The chosen slots in the order of expert, then slot: offsets by expert, the token of each row, the row of each slot; -1 where there is none."""
    t, k = ids.shape
    key = torch.where(ids < 0, experts, ids).reshape(-1)
    key, slot = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, dtype=key.dtype, device=key.device)).to(torch.int32)
    rows_of = torch.where(key < experts, slot // k, -1).to(torch.int32)
    at = torch.where(key < experts, torch.arange(t * k, device=key.device), -1).to(torch.int32)
    return offsets, rows_of, torch.empty_like(at).index_copy_(0, slot, at)


def _route(s):
    e, k, soft = s["experts"], s["top"], s["score"] == "softmax"
    l64 = s["logits"].double()  # two keys next to one another are told apart in 64 bits
    s64 = torch.softmax(l64, 1) if soft else torch.sigmoid(l64)
    biased = s64 if s["bias_of"] is None else s64 + s["bias_of"].double()
    key = l64 if s["bias_of"] is None else biased
    if s["groups"] > 1:
        best = biased.view(-1, s["groups"], e // s["groups"]).sort(dim=2, descending=True)[0][:, :, : s["best"]].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True)[1][:, : s["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True).repeat_interleave(e // s["groups"], 1)
        key = torch.where(keep, key, -math.inf)
    ids = key.sort(dim=1, descending=True, stable=True)[1][:, :k]
    logits = s["logits"].float()
    w = (torch.softmax(logits, 1) if soft else torch.sigmoid(logits)).gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = w * s["scale"]
    if s["live"] is not None:
        live = s["live"][:, None] != 0
        ids, w = torch.where(live, ids, -1), torch.where(live, w, 0.0)
    return ids.to(torch.int32), w


def _route_grad(s):
    logits, g, ids = s["logits"].float(), s["dweights"], s["ids"].long()
    chosen = torch.zeros_like(logits).scatter_(1, ids, 1.0)
    g = torch.zeros_like(logits).scatter_(1, ids, g)
    if s["score"] == "softmax":
        p = torch.softmax(logits, 1)
        if s["renorm"]:
            p = p * chosen
            p = p / p.sum(1, keepdim=True)
        d = p * (g - (g * p).sum(1, keepdim=True))
    else:
        p = torch.sigmoid(logits)
        back = torch.sigmoid(-logits)  # 1 - p
        if s["renorm"]:
            p = p * chosen
            p = p / p.sum(1, keepdim=True)
            g = g - (g * p).sum(1, keepdim=True)
        d = p * back * g
    return (d * s["scale"]).to(s["logits"].dtype)


def run(state):
    if own:
        return _own(state)
    s, op = state, state["op"]
    if op == "norm":
        h = s["x"].float() if s["res"] is None else s["x"].float() + s["res"].float()
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["w"].float()
        out = {"y": y.to(s["x"].dtype)} if s["y"] is not None else {}
        if s["res"] is not None:
            out["h"] = h.to(s["x"].dtype)
        if s["fmt"]:
            out["q"], out["s"] = _quantize(y, s["fmt"])
        return out
    if op == "norm_grad":
        h, dy = s["h"].float(), s["dy"].float()
        r = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
        a, n = dy * s["w"].float(), h * r
        dx = r * (a - n * (a * n).mean(1, keepdim=True))
        if s["dres"] is not None:
            dx = dx + s["dres"].float()
        return {"dx": dx.to(s["h"].dtype), "dw": (dy * n).sum(0)}
    if op == "route":
        ids, w = _route(s)
        offsets, rows_of, row_at = _order(ids, s["experts"])
        return {"ids": ids, "weights": w, "offsets": offsets, "rows_of": rows_of, "row_at": row_at}
    if op == "route_grad":
        return _route_grad(s)
    t, k = s["t"], s["top"]
    at = s["row_at"].long()
    if op == "combine":
        rows = s["rows"][at].float().view(t, k, -1)
        y = (rows if s["w"] is None else rows * s["w"][:, :, None]).sum(1)
        return (y if s["base_of"] is None else y + s["base_of"].float()).to(TYPES[s["ytype"]])
    dy = s["dy"].float()[:, None]
    drows = torch.empty_like(s["rows"]).index_copy_(0, at, (dy * s["w"][:, :, None]).to(s["rows"].dtype).view(t * k, -1))
    return {"drows": drows, "dweights": (s["rows"][at].float().view(t, k, -1) * dy).sum(2)}


# ── this framework's kernels ─────────────────────────────────────────────────
def _own(s):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mantle.jl_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mantle_cuda as M

    stream, op, k = torch.cuda.current_stream().cuda_stream, s["op"], M.kernels
    kind = TYPE[s["type"]]
    if op == "norm":
        M.launch(k.rms_norm, (s["y"], s["q"], s["s"], s["h"], s["x"], s["res"], s["w"], s["cols"], kind, TYPE[s["wtype"]],
                              FORMAT.get(s["fmt"], 0), 0, EPS), s["rows"], stream=stream)
        return {n: s[n] for n in ("y", "h", "q", "s") if s[n] is not None}
    if op == "norm_grad":
        args = (s["dx"], s["dw"], s["dy"], s["h"], s["w"], s["dres"], s["cols"], kind, TYPE[s["wtype"]], EPS)
        M.launch(k.rms_norm_grad, args, s["rows"], stream=stream, workspace=_scratch(M, s, k.rms_norm_grad, args, s["rows"]))
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "route":
        args = (s["ids"], s["weights"], s["offsets"], s["rows_of"], s["row_at"], s["logits"], s["bias_of"], s["live"], s["experts"], s["top"],
                s["groups"], s["top_groups"], s["best"], SCORE[s["score"]], int(s["renorm"]), kind, s["scale"])
        M.launch(k.route_experts, args, s["t"], stream=stream, workspace=_scratch(M, s, k.route_experts, args, s["t"]))
        return {n: s[n] for n in ("ids", "weights", "offsets", "rows_of", "row_at")}
    if op == "route_grad":
        M.launch(k.route_experts_grad, (s["dlogits"], s["dweights"], s["logits"], s["ids"], s["experts"], s["top"], SCORE[s["score"]],
                                        int(s["renorm"]), kind, s["scale"]), s["t"], stream=stream)
        return s["dlogits"]
    n = s["t"] * s["top"]
    if op == "combine":
        M.launch(k.combine_experts, (s["out"], s["rows"], s["w"], s["row_at"], s["base_of"], n, s["cols"], s["top"], kind, TYPE[s["ytype"]]),
                 s["t"], stream=stream)
        return s["out"]
    M.launch(k.combine_experts_grad, (s["drows"], s["dweights"], s["dy"], s["rows"], s["w"], s["row_at"], s["rows_of"], n, s["cols"], s["top"],
                                      kind, TYPE[s["ytype"]]), s["t"], stream=stream)
    return {"drows": s["drows"], "dweights": s["dweights"]}


def _scratch(M, s, kernel, args, ndrange):
    """The call's scratch, allocated once and kept beside its outputs."""
    if "scratch" not in s:
        size = M.workspace_bytes(kernel, args, ndrange)
        s["scratch"] = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    return s["scratch"]


# ── what a pass cannot do without ────────────────────────────────────────────
def work(case):
    op, per = case["op"], {"bf16": 2, "f32": 4}
    b = per[case["type"]]
    if op in ("norm", "norm_grad"):
        r, c, bw = case["rows"], case["cols"], per[case["wtype"]]
        if op == "norm_grad":
            return {"bytes": r * c * b * (4 if case["residual"] else 3) + c * (bw + 4), "flops": 12 * r * c}
        out = (r * _up(c, 16) + 4 * r * -(-c // 128)) if case["fmt"] else 0
        return {"bytes": r * c * b * (1 + 2 * case["residual"] + case["y"]) + out + c * bw, "flops": 5 * r * c}
    t, k = case["t"], case["top"]
    if op == "route":
        e = case["experts"]
        return {"bytes": t * e * b + 4 * e * (1 + case["bias"]) + 16 * t * k + 4 * t * case["padded"], "flops": 8 * t * e}
    if op == "route_grad":
        e = case["experts"]
        return {"bytes": 2 * t * e * b + 8 * t * k, "flops": 8 * t * e}
    c, by = case["cols"], per[case["ytype"]]
    if op == "combine":
        return {"bytes": t * k * (c * b + 4 + 4 * case["weighted"]) + t * c * by * (1 + case["base"]), "flops": 2 * t * k * c}
    return {"bytes": t * k * (2 * c * b + 16) + t * c * by, "flops": 3 * t * k * c}


# ── in 64 bits ───────────────────────────────────────────────────────────────
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    d = lambda n: s[n].double()  # noqa: E731
    if op == "norm":
        h = d("x") if s["res"] is None else d("x") + d("res")
        length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        y = h / torch.sqrt(length * length / case["cols"] + EPS) * d("w")
        out = {"y": y} if case["y"] else {}
        if case["residual"]:
            out["h"] = h
        if case["fmt"]:
            out["q"], out["s"] = _exact_codes(y, case["fmt"])
        return out
    if op == "norm_grad":
        h, dy, c = d("h"), d("dy"), case["cols"]
        var = (h * h).sum(1, keepdim=True) / c + EPS
        dot = (dy * d("w") * h).sum(1, keepdim=True)
        dx = dy * d("w") / var.sqrt() - h * dot / (c * var * var.sqrt())
        return {"dx": dx if s["dres"] is None else dx + d("dres"), "dw": ((dy * h) / var.sqrt()).sum(0)}
    if op == "route":
        return {"ids": None, "weights": _exact_weights(s), "offsets": None, "rows_of": None, "row_at": None}
    if op == "route_grad":
        l, g, ids = d("logits"), d("dweights"), s["ids"].long()
        out = torch.zeros_like(l)
        lse = torch.logsumexp(l, 1, keepdim=True)
        u = torch.exp(l.gather(1, ids) - lse) if case["score"] == "softmax" else 1 / (1 + torch.exp(-l.gather(1, ids)))
        if case["renorm"]:
            share = u / u.sum(1, keepdim=True)
            rest = g - (g * share).sum(1, keepdim=True)
            return out.scatter_(1, ids, share * rest * (1 if case["score"] == "softmax" else 1 - u)) * s["scale"]
        if case["score"] == "sigmoid":
            return out.scatter_(1, ids, g * u * (1 - u)) * s["scale"]
        out -= torch.exp(l - lse) * (g * u).sum(1, keepdim=True)
        return out.scatter_add_(1, ids, g * u) * s["scale"]
    t, k = case["t"], case["top"]
    at = s["row_at"].long().view(t, k)
    if op == "combine":
        y = torch.zeros((t, case["cols"]), dtype=torch.float64, device="cuda") if s["base_of"] is None else d("base_of")
        for j in range(k):
            y = y + s["rows"][at[:, j]].double() * (1.0 if s["w"] is None else s["w"][:, j, None].double())
        return y
    dy = d("dy")
    drows, dw = torch.zeros((t * k, case["cols"]), dtype=torch.float64, device="cuda"), []
    for j in range(k):
        drows[at[:, j]] = dy * s["w"][:, j, None].double()
        dw.append(torch.einsum("tc,tc->t", dy, s["rows"][at[:, j]].double()))
    return {"drows": drows, "dweights": torch.stack(dw, 1)}


def _exact_weights(s):
    """The chosen experts one after the other, each the lowest index of the largest key left; then their weights."""
    l, t, e, k = s["logits"].double(), s["t"], s["experts"], s["top"]
    index = torch.arange(e, device="cuda").expand(t, e)
    score = 1 / (1 + torch.exp(-l)) if s["score"] == "sigmoid" else torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    key = score if s["bias_of"] is None else score + s["bias_of"].double()
    per = e // s["groups"]
    if s["groups"] > 1:
        value = key.view(t, s["groups"], per).topk(s["best"], 2)[0].sum(2)
        number = torch.arange(s["groups"], device="cuda")
        ahead = (value[:, None] > value[:, :, None]) | ((value[:, None] == value[:, :, None]) & (number < number[:, None]))
        key = torch.where((ahead.sum(2) < s["top_groups"])[:, :, None], key.view(t, s["groups"], per), -math.inf).reshape(t, e)
    w = []
    for _ in range(k):
        at = torch.where(key == key.amax(1, keepdim=True), index, e).amin(1, keepdim=True)
        w.append(score.gather(1, at))
        key = key.scatter(1, at, -math.inf)
    w = torch.cat(w, 1)
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return w * s["scale"] * (1.0 if s["live"] is None else s["live"][:, None].double())


def _exact_codes(y, fmt):
    """The codes' values and the scales of y (rows, cols) in 64 bits; the roundings of the scale and its inverse to 32 bits are part of their definition."""
    r, c = y.shape
    block = torch.arange(c, device=y.device) // 128
    a = torch.full((r, int(block[-1]) + 1), SMALLEST, dtype=torch.float64, device=y.device)
    a.scatter_reduce_(1, block.expand(r, c), y.abs(), "amax")
    top = LARGEST[fmt]
    v = y * (top / a).float().double()[:, block]
    digits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low))) - digits)
    q = torch.zeros((r, _up(c, 16)), dtype=torch.float64, device=y.device)
    q[:, :c] = (torch.round(v / step) * step).clamp(-top, top)
    return q, (a / top).float().double().t()
