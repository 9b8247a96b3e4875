"""Routing to experts against a plain restatement in 64 bits: the choice and the rows'
order exactly, weights and gradients within the roundings of 32 bits.

u = 2^-24, D the largest difference of two logits of a token. exp of a difference is off by
2 units of its result (2 u each) and by u D from the rounded difference; a sum of positive
terms adds u for each of at most 37 additions, a quotient and the scale u each. A score is
thus off by (D + 4 + D + 4 + 37 + 3) u of itself at most, one over the chosen's sum by
less: (2 D + 64) u covers both, and so it does sigmoid's score (D replaced by |l|, whose
exp has no difference to round).

The gradient's factors are such scores, and 1 - s likewise; with e = (2 D + 64) u, and
S = |g| + sum |g| u, its terms are off by 4 e of c u S at most.
"""
import numpy as np
import pytest
import torch

import mantle_cuda as M

u = 2.0 ** -24
F, H = torch.float32, torch.bfloat16
SOFTMAX, SIGMOID = 0, 1
ptr = lambda n, at=1 << 20: M.DevicePtr(at, n)  # noqa: E731
BIG = ptr(1 << 40)


# ── the restatement ──────────────────────────────────────────────────────────
def scores(l, score):
    l = l.astype(np.float64)
    with np.errstate(all="ignore"):
        if score == SIGMOID:
            return 1 / (1 + np.exp(-l))
        m = l.max()
        if m == -np.inf:
            return np.zeros_like(l)
        p = np.exp(l - m)
        return p / p.sum()


def choose(l, top, score, bias=None, groups=1, top_groups=1, best=1):
    """The chosen experts of one token's logits, or None for a token that is not a number."""
    if np.isnan(l).any() or (bias is not None and np.isnan(bias).any()) or (score == SOFTMAX and l.max() == np.inf):
        return None
    s = scores(l, score)
    key = l.astype(np.float64) if bias is None else s + bias.astype(np.float64)
    for_groups = s if bias is None else key
    key, for_groups = (np.where(l == -np.inf, -np.inf, v) for v in (key, for_groups))
    E = len(l)
    if groups > 1:
        per = E // groups
        if bias is None and best == 1:
            for_groups = key
        value = np.array([sum(x for i, x in enumerate(sorted(for_groups[g * per:(g + 1) * per], reverse=True)[:best]) if i == 0 or x > -np.inf)
                          for g in range(groups)])
        keep = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
        key = np.array([key[e] if e // per in keep else -np.inf for e in range(E)])
    order = sorted(range(E), key=lambda e: (-key[e], e))[:top]
    return [e for e in order if key[e] > -np.inf]


def routed(logits, top, score, renorm, scale=1.0, bias=None, live=None, **groups):
    """ids (T, top) and weights (T, top) in 64 bits."""
    T = len(logits)
    ids, w = np.full((T, top), -1), np.zeros((T, top))
    for t in range(T):
        if live is not None and not live[t]:
            continue
        c = choose(logits[t], top, score, bias, **groups)
        if c is None:
            w[t] = np.nan
            continue
        if not c:
            continue
        ids[t, :len(c)] = c
        l = logits[t].astype(np.float64)
        if renorm:  # relative to the largest, so that no sum underflows
            if score == SOFTMAX:
                x = np.exp(l[c] - l[c].max())
            else:
                x = np.exp(np.minimum(l[c], 0) - min(l[c].max(), 0)) / (1 + np.exp(-np.abs(l[c])))
            w[t, :len(c)] = x / x.sum() * scale
        else:
            w[t, :len(c)] = scores(l, score)[c] * scale
    return ids, w


def ordered(ids, E):
    """offsets, rows_of, row_at of the chosen slots by expert, then slot."""
    T, top = ids.shape
    flat = ids.reshape(-1)
    rows = [s for e in range(E) for s in np.flatnonzero(flat == e)]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=E))])
    rows_of, row_at = np.full(T * top, -1), np.full(T * top, -1)
    rows_of[:len(rows)] = np.array(rows, dtype=int) // top
    row_at[rows] = np.arange(len(rows))
    return offsets, rows_of, row_at


def test_the_restatement():
    l = np.array([[1.0, 3.0, 3.0, -np.inf, 2.0, 0.0]], np.float32)
    assert routed(l, 3, SOFTMAX, True)[0].tolist() == [[1, 2, 4]]
    assert routed(l, 6, SOFTMAX, False)[0].tolist() == [[1, 2, 4, 0, 5, -1]]
    assert routed(l, 2, SIGMOID, True, bias=np.array([1, 0, 0, 9, 0, 0.9]))[0].tolist() == [[0, 5]]
    assert routed(l, 2, SIGMOID, True, groups=3, top_groups=1)[0].tolist() == [[1, 0]]  # groups 0 and 1 tie
    assert ordered(np.array([[1, 0], [-1, 1]]), 3)[1].tolist() == [0, 0, 1, -1]


# ── refusals (no launch) ─────────────────────────────────────────────────────
def r_args(t=4, E=8, top=2, groups=1, top_groups=1, best=1, score=0, renorm=0, kind=0, scale=1.0, **change):
    n = 4 * t * top
    a = dict(ids=ptr(n), w=ptr(n), off=ptr(4 * (E + 1)), rows=ptr(n), at=ptr(n), l=ptr(t * E * (2 if kind == 1 else 4)), bias=None, live=None)
    a.update(change)
    return [*a.values(), E, top, groups, top_groups, best, score, renorm, kind, scale]


@pytest.mark.parametrize("args,nd,match", [
    (r_args(ids=ptr(31)), 4, "ids"), (r_args(w=ptr(31)), 4, "the weights"), (r_args(off=ptr(35)), 4, "offsets"),
    (r_args(rows=ptr(31)), 4, "rows_of"), (r_args(at=ptr(31)), 4, "row_at"), (r_args(l=ptr(127)), 4, "the logits"),
    (r_args(kind=1, l=ptr(63)), 4, "the logits"), (r_args(bias=ptr(31)), 4, "the bias"), (r_args(live=ptr(15)), 4, "live"),
    (r_args(), 5, "ids"), (r_args(off=None), 4, "go together"), (r_args(rows=None), 4, "go together"), (r_args(at=None), 4, "go together"),
    (r_args(top=0), 4, "top must be"), (r_args(top=9), 4, "top must be"), (r_args(E=64, top=33), 4, "top must be"),
    (r_args(E=0), 4, "no experts"), (r_args(E=1025), 4, "more than 1024 experts"),
    (r_args(groups=3), 4, "divide the experts"), (r_args(groups=0), 4, "divide the experts"), (r_args(groups=16), 4, "divide the experts"),
    (r_args(groups=4, top_groups=5), 4, "top_groups"), (r_args(groups=4, top_groups=0), 4, "top_groups"),
    (r_args(groups=4, best=3), 4, "best two"), (r_args(groups=8, best=2), 4, "best two"), (r_args(best=0), 4, "best two"),
    (r_args(score=2), 4, "must be 0 or 1"), (r_args(renorm=-1), 4, "must be 0 or 1"), (r_args(kind=2), 4, "must be 0 or 1"),
    (r_args(scale=float("nan")), 4, "finite"), (r_args(scale=float("inf")), 4, "finite"),
    (r_args(ids=BIG, w=BIG, rows=BIG, at=BIG, l=BIG), 1 << 30, "slots"), (r_args(), (4, 1), "one-dimensional"),
    (r_args(l=ptr(1 << 20, (1 << 20) + 2)), 4, "4-byte aligned"), (r_args(bias=ptr(0, 0)), 4, "the bias must be a device buffer"),
    (r_args(live=ptr(0, 0)), 4, "live must be a device buffer"), (r_args(ids=ptr(0, 0)), 4, "ids must be a device buffer"),
])
def test_route_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.route_experts, args, nd)


def d_args(t=4, E=8, top=2, score=0, renorm=0, kind=0, scale=1.0, **change):
    per = 2 if kind == 1 else 4
    a = dict(dl=ptr(t * E * per), dw=ptr(4 * t * top), l=ptr(t * E * per), ids=ptr(4 * t * top))
    a.update(change)
    return [*a.values(), E, top, score, renorm, kind, scale]


@pytest.mark.parametrize("args,nd,match", [
    (d_args(dl=ptr(127)), 4, "dlogits"), (d_args(dw=ptr(31)), 4, "the weights' gradient"), (d_args(l=ptr(127)), 4, "the logits"),
    (d_args(ids=ptr(31)), 4, "ids"), (d_args(), 5, "dlogits"), (d_args(top=9), 4, "top must be"), (d_args(score=3), 4, "must be 0 or 1"),
    (d_args(renorm=3), 4, "must be 0 or 1"), (d_args(kind=3), 4, "must be 0 or 1"), (d_args(scale=float("inf")), 4, "finite"),
    (d_args(E=2000), 4, "more than 1024"), (d_args(ids=ptr(0, 0)), 4, "ids must be a device buffer"),
])
def test_route_grad_refuses(args, nd, match):
    with pytest.raises(M.MantleError, match=match):
        M.launch(M.kernels.route_experts_grad, args, nd)


# ── on the device ────────────────────────────────────────────────────────────
def stream():
    return torch.cuda.current_stream().cuda_stream


def route(logits, top, score, renorm, scale=1.0, bias=None, live=None, groups=1, top_groups=1, best=1, order=True):
    T, E = logits.shape
    i = lambda n: torch.full((n,), -7, dtype=torch.int32, device="cuda")  # noqa: E731
    ids, w = i(T * top), torch.full((T * top,), -7.0, device="cuda")
    rest = (i(E + 1), i(T * top), i(T * top)) if order else (None, None, None)
    args = (ids, w, *rest, logits, bias, live, E, top, groups, top_groups, best, score, renorm, int(logits.dtype == H), scale)
    need = M.workspace_bytes(M.kernels.route_experts, args, T)
    M.launch(M.kernels.route_experts, args, T, stream=stream(), workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
    torch.cuda.synchronize()
    return ids.view(T, top), w.view(T, top), rest


def check(logits, top, score, renorm, scale=1.0, bias=None, live=None, **groups):
    ids, w, rest = route(logits.cuda(), top, score, renorm, scale, None if bias is None else bias.cuda(), None if live is None else live.cuda(), **groups)
    l = logits.float().numpy()
    want, weights = routed(l, top, score, renorm, scale, None if bias is None else bias.numpy(), None if live is None else live.numpy(), **groups)
    assert np.array_equal(ids.cpu().numpy(), want)
    got = w.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(weights))
    fine = ~np.isnan(weights)
    with np.errstate(invalid="ignore"):
        finite = np.where(np.isfinite(l), l, 0).astype(np.float64)
        D = (finite.max(1) - finite.min(1) + np.abs(finite).max(1))[:, None] * np.ones((1, top))
    assert (np.abs(got - weights)[fine] <= ((2 * D + 64) * u * np.abs(weights) + 1e-44)[fine]).all()
    for a, b in zip(rest, ordered(want, logits.shape[1])):
        assert np.array_equal(a.cpu().numpy(), b)
    alone = route(logits.cuda(), top, score, renorm, scale, None if bias is None else bias.cuda(), None if live is None else live.cuda(), order=False, **groups)
    assert torch.equal(alone[0], ids) and torch.equal(alone[1].nan_to_num(9), w.nan_to_num(9))


def normal(*shape, seed=0, kind=F):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(kind)


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 7, 3), (33, 32, 4), (70, 64, 6), (3, 100, 32), (31, 160, 6), (257, 256, 8), (9, 384, 8), (12, 1000, 5), (4, 1024, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("t,e,top", SHAPES)
def test_route(dev, t, e, top, score, renorm, kind):
    l = 2 * normal(t, e, seed=t, kind=kind)  # in bfloat16 many logits are equal
    check(l, top, score, renorm)
    check(l, top, score, renorm, 2.5, bias=0.1 * normal(e, seed=3))
    check(l, top, score, renorm, bias=torch.zeros(e))
    check(l, top, score, renorm, -0.5, live=(torch.arange(t) % 3 != 1).to(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("t,e,top,groups,top_groups,best", [
    (40, 256, 8, 8, 4, 2), (40, 64, 6, 8, 3, 1), (33, 160, 6, 8, 3, 1), (20, 96, 4, 6, 2, 2), (7, 16, 2, 16, 4, 1), (9, 1024, 8, 32, 5, 2),
    (5, 1024, 8, 1024, 9, 1), (5, 1000, 8, 200, 3, 2), (6, 8, 8, 4, 2, 2), (50, 256, 8, 4, 4, 2), (40, 148, 5, 4, 2, 2),
    (9, 1023, 7, 31, 4, 2), (9, 992, 7, 31, 4, 1), (30, 33, 3, 11, 3, 2), (12, 24, 2, 3, 1, 1)])
def test_route_in_groups(dev, t, e, top, groups, top_groups, best, score, kind):
    g = dict(groups=groups, top_groups=top_groups, best=best)
    l = 2 * normal(t, e, seed=e, kind=kind)
    check(l, top, score, 1, **g)
    check(l, top, score, 0, 2.5, bias=0.1 * normal(e, seed=3), **g)
    l[::2, : e // groups] = float("-inf")  # a whole group masked
    l[1::2, ::2] = float("-inf")
    check(l, top, score, 1, bias=0.1 * normal(e, seed=4), **g)
    check(l, top, score, 1, **g)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("bias", [False, True])
def test_masks_and_values_that_are_not_numbers(dev, score, bias):
    inf, nan = float("inf"), float("nan")
    l = normal(12, 40)
    l[0] = -inf                      # nothing left
    l[1, 3:] = -inf                  # fewer than asked for
    l[2, 7] = nan
    l[3] = nan
    l[4, 9] = inf                    # first under sigmoid, no number under softmax
    l[5] = -3.0e38                   # the type's lowest values
    l[6] = torch.where(torch.arange(40) % 2 == 0, -3.4e38, -inf)
    l[7] = 0
    l[8, :20], l[8, 20:] = 3.4e38, -3.4e38
    l[9] = -200.0                    # scores that are zeros in 32 bits
    l[9, 5] = -199.0
    l[10, 0], l[10, 1] = 0.0, -0.0
    b = None if not bias else 0.01 * normal(40, seed=2)
    for renorm in (0, 1):
        check(l, 6, score, renorm, bias=b)
        check(l, 6, score, renorm, bias=b, groups=5, top_groups=2, best=2)
        if bias:
            b2 = b.clone()
            b2[:36] = -inf
            check(l[[5, 7, 10, 11]], 6, score, renorm, bias=b2)
            b2[0] = nan
            check(l[[5, 7, 10, 11]], 6, score, renorm, bias=b2)
    # dead tokens count for nothing, whatever they hold
    check(l, 6, score, 1, bias=b, live=torch.zeros(12, dtype=torch.int32))


@pytest.mark.gpu
def test_keys_that_32_bits_do_not_tell_apart(dev):
    # scores plus biases that are equal or next to one another in 32 bits, and not in 64
    E, T = 64, 40
    l = normal(1, E, seed=1).expand(T, E).clone()
    s = torch.sigmoid(l[0].double())
    b = (0.75 - s).float()  # every key 0.75 but for the bias's own rounding, 2^-25 at most
    for t in range(T):
        l[t, t] += 2e-7
    check(l, 8, SIGMOID, 1, bias=b)
    check(l, 8, SIGMOID, 1, bias=b, groups=8, top_groups=3, best=2)
    p = torch.softmax(l[0].double(), 0)
    check(l, 8, SOFTMAX, 0, bias=(0.03 - p).float())
    check(l, 8, SOFTMAX, 0, bias=(0.03 - p).float(), groups=4, top_groups=2, best=1)


def near_pairs(score, n, seed):
    """Two logits, and a bias of the second in 32 bits, whose keys s(x) and s(x2) + bias are (3.2 .. 32) 1e-15 of s(x) apart;
    and which is larger, told in 80 bits. For softmax there is a third logit, the largest, which the bias excludes."""
    r, wide = np.random.default_rng(seed), np.longdouble
    if score == SIGMOID:
        x = np.where(r.random(n) < 0.3, r.uniform(-1, 12, n), r.uniform(-60, 1, n)).astype(np.float32)
        s = lambda v: 1 / (1 + np.exp(-v.astype(wide)))  # noqa: E731
        slope = s(-x)  # of s, by s
        m = np.zeros(n, np.float32)
    else:
        m = r.uniform(0, 5, n).astype(np.float32)
        x = (m - r.uniform(0.01, 60, n)).astype(np.float32)
    step = 3e-7 * r.uniform(0.3, 3, n)
    if score == SIGMOID:
        x2 = np.minimum((x - step / slope.astype(np.float64)).astype(np.float32), np.nextafter(x, np.float32(-np.inf)))
        a, c = s(x), s(x2)
    else:
        x2 = np.minimum((x - step).astype(np.float32), np.nextafter(x, np.float32(-np.inf)))
        e = [np.exp(v.astype(wide) - m.astype(wide)) for v in (m, x, x2)]
        a, c = e[1] / sum(e), e[2] / sum(e)
    b = (a - c).astype(np.float32)
    apart = (a - (c + b.astype(wide))) / a
    near = (np.abs(apart) > 3.2e-15) & (np.abs(apart) < 3.2e-14) & (b > 1e-37)
    return x[near], x2[near], b[near], m[near], apart[near] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_scores_hold_in_64_bits(dev, score):
    # An exponential is off by 1e-15 of itself at most; a score has three roundings more and the sum with its bias one, of
    # 1.1e-16 each: two keys are off by (2 * (1e-15 + 3.3e-16) + 2.2e-16) of the larger score together, below 3.2e-15.
    x, x2, b, m, first = near_pairs(score, 60000, 1)
    n = min(len(x), 1500)
    assert n > 500 and 0.3 < first[:n].mean() < 0.7
    lowest = np.float32(-np.inf) if score == SIGMOID else None
    swap = np.arange(n) % 2 == 1  # either may have the lower index
    l, bias = np.zeros((n, 3), np.float32), np.zeros((n, 3), np.float32)
    l[:, 0], bias[:, 0] = (lowest if lowest is not None else m[:n]), -1.0
    l[:, 1], l[:, 2] = np.where(swap, x2[:n], x[:n]), np.where(swap, x[:n], x2[:n])
    bias[:, 1], bias[:, 2] = np.where(swap, b[:n], 0), np.where(swap, 0, b[:n])
    L, B = torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda()
    ids, w = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    for i in range(n):
        M.launch(M.kernels.route_experts, (ids[i:i + 1], w[i:i + 1], None, None, None, L[i:i + 1], B[i], None, 3, 1, 1, 1, 1, score, 0, 0, 1.0), 1, stream=stream())
    want = np.where(first[:n] != swap, 1, 2)
    assert np.array_equal(ids.cpu().numpy(), want)


@pytest.mark.gpu
def test_scores_that_are_denormal_in_64_bits(dev):
    # groups' values are sums of scores: of -700 and below they are denormal, down to the smallest, and then zeros
    a = np.array([-1, -87, -104, -650, -708, -709, -720, -730, -740, -743, -744], np.float32)
    pairs = [(p, q) for p in a for q in a if p != q]
    l = np.full((len(pairs), 4), -np.inf, np.float32)
    l[:, 0], l[:, 2] = np.array(pairs).T
    ids, _, _ = route(torch.from_numpy(l).cuda(), 1, SIGMOID, 0, groups=2, top_groups=1, best=2)
    assert np.array_equal(ids.cpu().numpy()[:, 0], np.where(l[:, 0] > l[:, 2], 0, 2))
    l[:, 0], l[:, 2] = -800, -750
    ids, _, _ = route(torch.from_numpy(l).cuda(), 1, SIGMOID, 0, groups=2, top_groups=1, best=2)
    assert (ids == 0).all()  # both zeros, and so the lower group


@pytest.mark.gpu
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_biases_that_are_large_or_infinite(dev, score):
    l = normal(130, 48, seed=3)
    b = 0.05 * normal(48, seed=4)
    for change in ({3: float("inf")}, {3: float("inf"), 40: float("inf")}, {5: float("-inf"), 6: float("inf")}, {i: 1e30 for i in range(0, 48, 2)},
                   {i: 4096.0 for i in range(10)}, {i: -3e38 for i in range(44)}):
        x = b.clone()
        for i, v in change.items():
            x[i] = v
        check(l, 6, score, 1, bias=x)
        check(l, 6, score, 0, bias=x, groups=4, top_groups=2, best=2)
        check(l, 6, score, 0, bias=x, groups=4, top_groups=2, best=1)
    check(l, 32, score, 1, bias=b)  # a slot for every lane
    check(l.to(H), 32, score, 1, bias=torch.zeros(48))  # and many ties
    check(torch.zeros(5, 700), 32, score, 1, bias=torch.zeros(700))  # more equal keys than lanes
    check(torch.zeros(5, 700), 32, score, 1, bias=torch.zeros(700), groups=7, top_groups=3, best=2)
    check(torch.zeros(5, 700), 32, score, 1, groups=7, top_groups=3, best=2)
    check(torch.zeros(5, 256), 8, score, 1, bias=torch.zeros(256), groups=8, top_groups=3, best=2)
    check(torch.zeros(5, 256), 8, score, 1, bias=torch.zeros(256), groups=8, top_groups=3, best=1)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [32, 33, 127, 128, 129, 1023, 1025])
def test_few_tokens_and_many_are_one(dev, t):
    # one launch or two, one cluster or several: the same, token by token
    l, b = normal(t, 40, seed=1), 0.1 * normal(40, seed=2)
    check(l, 5, SIGMOID, 1, 2.5, bias=b, groups=5, top_groups=3, best=2)
    live = (torch.arange(t) % 5 != 2).to(torch.int32)
    check(l, 5, SOFTMAX, 0, live=live)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("t", [1, 16, 17, 96, 128, 129])
@pytest.mark.parametrize("e,groups", [(1, 1), (32, 4), (33, 1), (60, 3), (64, 64), (65, 5), (128, 8), (129, 1), (256, 8), (256, 256), (640, 1), (1024, 8)])
def test_a_captured_call_gives_what_a_direct_one_does(dev, t, e, groups, kind):
    # whose launches differ: a direct call of few tokens and experts is one kernel, a captured one two
    l, b, top = normal(t, e, seed=t, kind=kind).cuda(), (0.1 * normal(e, seed=2)).cuda(), min(6, e // groups)
    g = dict(groups=groups, top_groups=max(1, groups // 2), best=min(2, e // groups))
    check(l.cpu(), top, SIGMOID, 1, bias=b.cpu(), **g)
    want = route(l, top, SIGMOID, 1, bias=b, **g)
    out = [torch.full((n,), -7, dtype=d, device="cuda") for n, d in ((t * top, torch.int32), (t * top, F), (e + 1, torch.int32), (t * top, torch.int32), (t * top, torch.int32))]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.launch(M.kernels.route_experts, (*out, l, b, None, e, top, groups, g["top_groups"], g["best"], SIGMOID, 1, int(kind == H), 1.0), t, stream=stream())
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, (want[0], want[1], *want[2])):
        assert torch.equal(x, y.reshape(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("t,e", [(1, 8), (64, 32), (128, 64), (60, 1024), (3000, 64)])
def test_a_replay_routes_in_two_kernels(dev, t, e):
    # few tokens too: one cluster for both takes a GPU longer, and a replay spares the host nothing
    L, n = M.Buffer.wrap(dev, normal(t, e).cuda(), dtype=np.float32), t * 2
    ids, rows_of, row_at, off, w = (M.Buffer(dev, d, k) for d, k in ((np.int32, n), (np.int32, n), (np.int32, n), (np.int32, e + 1), (np.float32, n)))
    g = M.Graph(dev)
    R, W = (lambda p, b: M.use(p, b, read=True)), (lambda p, b: M.use(p, b, write=True))
    M.compute(g, "route", lambda p: M.dispatch(p, M.kernels.route_experts, (
        W(p, ids), W(p, w), W(p, off), W(p, rows_of), W(p, row_at), R(p, L), None, None, e, 2, 1, 1, 1, 0, 1, 0, 1.0), t))
    plan = M.Plan(g)
    M.run(plan)
    dev.synchronize()
    assert plan.nkernels() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,top", [(0, 8, 2), (1, 1, 1), (3000, 8, 2), (2049, 16, 8), (1500, 300, 32), (9000, 1024, 2), (40000, 256, 8), (70000, 3, 1)])
def test_rows_in_order(dev, t, e, top):
    # slots in order within an expert, experts of very different sizes, some empty, and dead tokens between
    l = normal(t, e, seed=t) + torch.linspace(0, 4, e)
    live = (normal(t, seed=5) < 1).to(torch.int32)
    ids, w, rest = route(l.cuda(), top, SOFTMAX, 1, live=live.cuda())
    ids = ids.cpu().numpy()
    assert ((ids >= 0).all(1) == (live.numpy() != 0)).all() and (ids < e).all()
    for a, b in zip(rest, ordered(ids, e)):
        assert np.array_equal(a.cpu().numpy(), b)


def grad(logits, ids, g, score, renorm, scale):
    T, E = logits.shape
    dl = torch.full_like(logits, float("nan"))
    M.launch(M.kernels.route_experts_grad, (dl, g, logits, ids, E, ids.shape[1], score, renorm, int(logits.dtype == H), scale), T, stream=stream())
    torch.cuda.synchronize()
    return dl


def exact_grad(l, ids, g, score, renorm, scale):
    """(gradient, the magnitudes that its roundings go by) in 64 bits, of torch tensors."""
    l, g = l.double(), g.double()
    valid = ids >= 0
    at, g = ids.clamp(min=0).long(), torch.where(valid, g, 0.0)
    s = torch.softmax(l, 1).nan_to_num() if score == SOFTMAX else torch.sigmoid(l)
    c = torch.where(valid, s.gather(1, at), 0.0)
    if renorm:
        c = c / c.sum(1, keepdim=True).clamp(min=1e-300)
    mean = (g * c).sum(1, keepdim=True) if renorm or score == SOFTMAX else torch.zeros(len(l), 1, dtype=torch.float64)
    most = (g.abs() * c).sum(1, keepdim=True)
    d, m = c * (g - mean), c * (g.abs() + most)
    if score == SIGMOID:
        rest = torch.sigmoid(-l).gather(1, at)
        d, m = d * rest, m * rest
    out, mag = torch.zeros_like(l), torch.zeros_like(l)
    if score == SOFTMAX and not renorm:
        out, mag = -s * mean, s * most
        d = c * g
    return scale * out.scatter_add(1, at, torch.where(valid, d, 0.0)), abs(scale) * mag.scatter_add(1, at, torch.where(valid, m, 0.0))


def check_grad(l, ids, g, score, renorm, scale):
    dl = grad(l.cuda(), ids.cuda(), g.cuda(), score, renorm, scale).double().cpu()
    want, mag = exact_grad(l, ids, g, score, renorm, scale)
    finite = torch.where(l.double().isfinite(), l.double(), 0.0)
    D = (finite.amax(1) - finite.amin(1) + finite.abs().amax(1))[:, None]
    tol = 4 * (2 * D + 64) * u * mag + 1e-40
    assert ((dl - want).abs() <= tol + (2.0 ** -8 if l.dtype == H else u) * (want.abs() + tol)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("t,e,top", SHAPES)
def test_route_grad(dev, t, e, top, score, renorm, kind):
    l, g = 2 * normal(t, e, seed=t, kind=kind), normal(t, top, seed=9)
    ids = l.float().argsort(1, descending=True)[:, :top].to(torch.int32)
    check_grad(l, ids, g, score, renorm, 1.0)
    ids[::2, top // 2:] = -1
    check_grad(l, ids, g, score, renorm, -2.5)
    if e > 1:
        l[1::2, 0] = float("-inf")
        ids = torch.where(l.gather(1, ids.clamp(min=0).long()) == float("-inf"), -1, ids)
        check_grad(l, ids.to(torch.int32), g, score, renorm, 1.0)
    check_grad(l, torch.full_like(ids, -1), g, score, renorm, 1.0)
    same = torch.zeros_like(ids) + e - 1  # one expert in every slot: the slots' gradients together
    check_grad(l, same.to(torch.int32), g, score, renorm, 1.0)
    for way in ((l, ids.to(torch.int32)), (l.to(F), torch.zeros_like(ids).to(torch.int32))):  # over the logits themselves
        x, i = way[0].cuda(), way[1].cuda()
        want = grad(x, i, g.cuda(), score, renorm, 1.5)
        M.launch(M.kernels.route_experts_grad, (x, g.cuda(), x, i, e, top, score, renorm, int(x.dtype == H), 1.5), t, stream=stream())
        # (rows whose chosen experts are masked, every one, are 0 / 0 over their sum)
        assert torch.equal(x.nan_to_num(9), want.nan_to_num(9))
    outside = torch.full((t, top), e, dtype=torch.int32)
    assert torch.equal(grad(l.cuda(), outside.cuda(), g.cuda(), score, renorm, 1.0), torch.zeros_like(l).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F, H])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("e", [5, 64, 300])
def test_tokens_without_experts_have_no_gradient(dev, e, score, renorm, kind):
    # padding whose logits were never set: the forward pass counts it for nothing, and so does this
    inf, nan = float("inf"), float("nan")
    l, g, top = 2 * normal(12, e, seed=e, kind=kind), normal(12, 3, seed=9), 3
    ids = l.float().argsort(1, descending=True)[:, :top].to(torch.int32)
    want = grad(l.cuda(), ids.cuda(), g.cuda(), score, renorm, 2.5)
    bad = l.clone()
    bad[0], bad[2, e - 1], bad[4], bad[6, 1], bad[8], bad[10] = nan, nan, inf, inf, -inf, 3.0e38
    ids[::2], g[::4] = -1, nan
    ids[2], ids[6] = e, -7  # outside the experts, as good as none
    got = grad(bad.cuda(), ids.cuda(), g.cuda(), score, renorm, 2.5)
    assert (got[::2] == 0).all() and torch.equal(got[1::2], want[1::2])
    # what the forward pass makes of such tokens, live or not
    live = torch.ones(12, dtype=torch.int32)
    live[::2] = 0
    for alive in (live, None):
        chosen, w, _ = route(bad.cuda(), top, score, renorm, live=None if alive is None else alive.cuda())
        none = (chosen < 0).all(1).cpu()
        assert none[:10:2].all() if alive is not None else none[8]
        d = grad(bad.cuda(), chosen, torch.ones(12, top, device="cuda"), score, renorm, 1.0)
        assert (d[none.cuda()] == 0).all() and d.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_route_grad_against_differences(dev, score, renorm):
    # 64-bit central differences of sum(g w) with a step of 1e-5, at ids held still
    l, g, e = normal(2, 12, seed=1), normal(2, 4, seed=2), 1e-5
    ids = l.argsort(1, descending=True)[:, :4]

    def loss(x):
        s = torch.softmax(x, 1) if score == SOFTMAX else torch.sigmoid(x)
        w = s.gather(1, ids)
        return (g.double() * (w / w.sum(1, keepdim=True) if renorm else w)).sum().item() * 1.5

    dl = grad(l.cuda(), ids.to(torch.int32).cuda(), g.cuda(), score, renorm, 1.5)
    for t in range(2):
        for i in range(12):
            step = torch.zeros(2, 12, dtype=torch.float64)
            step[t, i] = e
            assert abs((loss(l.double() + step) - loss(l.double() - step)) / (2 * e) - dl[t, i].item()) < 1e-5


@pytest.mark.gpu
def test_types_are_refused(dev):
    l = normal(4, 8).cuda()
    ids, w = torch.empty((4, 2), dtype=torch.int32, device="cuda"), torch.empty((4, 2), device="cuda")
    go = lambda i, ww, ll, kind=0, bias=None, live=None: M.launch(M.kernels.route_experts, (  # noqa: E731
        i, ww, None, None, None, ll, bias, live, 8, 2, 1, 1, 1, 0, 0, kind, 1.0), 4, stream=stream())
    go(ids, w, l)
    for args, match in (((ids.long(), w, l), "expected Int32"), ((ids, w.to(H), l), "expected Float32"), ((ids, w, l.to(H)), "expected Float32"),
                        ((ids, w, l, 1), "expected bfloat16"), ((ids, w, l, 0, l[0].to(H).contiguous()), "expected Float32"),
                        ((ids, w, l, 0, None, torch.ones(4, dtype=torch.bool, device="cuda")), "expected Int32"),
                        ((ids, w, l.t().contiguous().t()), "contiguous")):
        with pytest.raises(M.ArgumentError, match=match):
            go(*args)


@pytest.mark.gpu
def test_captured_and_at_once(dev):
    l = normal(3000, 64).cuda()
    want = route(l, 4, SOFTMAX, 1)
    fresh = lambda: (torch.zeros(12000, dtype=torch.int32, device="cuda"), torch.zeros(12000, device="cuda"),  # noqa: E731
                     *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (65, 12000, 12000)))
    args = lambda o: (*o, l, None, None, 64, 4, 1, 1, 1, 0, 1, 0, 1.0)  # noqa: E731
    need = M.workspace_bytes(M.kernels.route_experts, args(fresh()), 3000)
    scratch = lambda: torch.empty(need, dtype=torch.uint8, device="cuda") if need else None  # noqa: E731
    outs, graphs, sides, kept = [fresh(), fresh()], [], [torch.cuda.Stream() for _ in range(2)], [scratch(), scratch()]
    torch.cuda.synchronize()
    for o, side, ws in zip(outs, sides, kept):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            M.launch(M.kernels.route_experts, args(o), 3000, stream=stream(), workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0].view(3000, 4), want[0]) and torch.equal(o[1].view(3000, 4), want[1])
        assert all(torch.equal(a, b) for a, b in zip(o[2:], want[2]))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [60, 3000])
def test_as_a_plan(dev, t):
    E, top = 64, 4
    l = normal(t, E).cuda()
    want = route(l, top, SIGMOID, 1, 2.5, groups=8, top_groups=4, best=2)
    L, n = M.Buffer.wrap(dev, l, dtype=np.float32), t * top
    ids, rows_of, row_at, off, w = (M.Buffer(dev, d, k) for d, k in ((np.int32, n), (np.int32, n), (np.int32, n), (np.int32, E + 1), (np.float32, n)))
    dw, dl = M.Buffer(dev, normal(t, top, seed=2).numpy().reshape(-1)), M.Buffer(dev, np.float32, t * E)
    g = M.Graph(dev)
    R, W = (lambda p, b: M.use(p, b, read=True)), (lambda p, b: M.use(p, b, write=True))
    M.compute(g, "route", lambda p: M.dispatch(p, M.kernels.route_experts, (
        W(p, ids), W(p, w), W(p, off), W(p, rows_of), W(p, row_at), R(p, L), None, None, E, top, 8, 4, 2, 1, 1, 0, 2.5), t))
    alone = M.Plan(g)
    M.compute(g, "grad", lambda p: M.dispatch(p, M.kernels.route_experts_grad, (
        W(p, dl), R(p, dw), R(p, L), R(p, ids), E, top, 1, 1, 0, 2.5), t))
    both = M.Plan(g)
    for plan in (alone, both, both):
        M.run(plan)
    dev.synchronize()
    for a, b in zip((ids, w, off, rows_of, row_at), (want[0], want[1], *want[2])):
        assert np.array_equal(a.array(), b.cpu().numpy().reshape(-1))
    d = grad(l, want[0], torch.from_numpy(dw.array()).view(t, top).cuda(), SIGMOID, 1, 2.5)
    assert np.array_equal(dl.array(), d.cpu().numpy().reshape(-1))
