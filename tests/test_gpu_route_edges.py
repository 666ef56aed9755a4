"""Routing where scores, biases or logits leave the ordinary range: indices against the definition in 64 bits."""
import math

import pytest
import torch

from agillm41_b200 import ops
from oracle import route_oracle as ro

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
LOWEST = torch.finfo(torch.float32).min


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(n, E, seed=0, dtype=torch.float32):
    return (torch.randn(n, E, generator=gen(seed), device="cuda") * 1.5).to(dtype)


# (experts, k, groups, kept): both kernels, E on both sides of 32, k on both sides of 8, group counts that are and
# are not powers of two
SHAPES = [(14, 2, 1, 1), (24, 4, 3, 2), (24, 8, 4, 2), (64, 8, 1, 1), (64, 4, 8, 4), (64, 12, 8, 4), (96, 6, 3, 2),
          (256, 8, 1, 1), (256, 8, 8, 4), (256, 12, 1, 1)]


@pytest.mark.parametrize("E,k,groups,keep", SHAPES)
@pytest.mark.parametrize("biased", [False, True])
def test_nan_and_inf_logits_leave_the_others_alone(E, k, groups, keep, biased):
    """Under softmax too, a NaN logit takes out its own expert only, +inf is the limit of a large logit, and the
    row's weights are NaN, which the experts pass on."""
    n = 12
    x = make(n, E, E + k)
    x[1, 3] = NAN
    x[2, E - 1] = NAN
    x[2, :E // 2:3] = NAN
    x[3, 5] = INF
    x[4, 1] = x[4, E - 2] = INF
    x[5, 2], x[5, 7] = INF, NAN
    x[6, 4], x[6, 0] = NAN, -INF
    b = torch.randn(E, generator=gen(1), device="cuda") * 0.1 if biased else None
    for score in ("softmax", "sigmoid"):
        idx, w = ops.route_experts(x, k, score=score, bias=b, n_groups=groups, top_groups=keep)
        assert torch.equal(idx.long(), ro.choose(x, k, score, b, groups, keep))
        odd = torch.isnan(x).any(1) | ((x == INF).any(1) if score == "softmax" else False)
        assert torch.equal(torch.isnan(w).all(1), odd) and torch.equal(torch.isnan(w).any(1), odd)
        d, H = 64, 128
        w1 = ops.quantize_fp8_weight(torch.randn(E, H, d, generator=gen(2), device="cuda"))
        w2 = ops.quantize_fp8_weight(torch.randn(E, d, H, generator=gen(3), device="cuda"))
        y = ops.moe_experts_fp8(torch.ones(n, d, device="cuda", dtype=torch.bfloat16), idx, w, w1,
                                torch.zeros(E, H, device="cuda"), w2, torch.zeros(E, d, device="cuda"))
        assert torch.equal(torch.isnan(y).all(1), odd) and torch.equal(torch.isnan(y).any(1), odd)


# (experts, groups, kept)
GROUPS = [(32, 8, 3), (64, 8, 4), (64, 32, 3), (60, 30, 3), (48, 3, 2), (256, 8, 4), (512, 16, 4)]


@pytest.mark.parametrize("E,groups,keep", GROUPS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinite_biases_force_experts(E, groups, keep, score):
    """A bias of +inf puts its expert, and its group, before every finite one; equal ones go by index."""
    x = make(40, E, E)
    size = E // groups
    none = torch.zeros(E, device="cuda")
    pair, each, some, far = none.clone(), none.clone(), none.clone(), none.clone()
    pair[:2] = INF                                   # two in one group
    each[::size] = INF                               # one in every group
    some[size - 1:size + 1] = some[E - 1] = INF      # three in three groups
    far[E - size:E - size + 2] = INF
    far[0] = -INF
    for bias in (pair, each, some, far):
        for k in (2, 6, 8, 9):
            idx, w = ops.route_experts(x, k, score=score, bias=bias, n_groups=groups, top_groups=keep)
            assert torch.equal(idx.long(), ro.choose(x, k, score, bias, groups, keep))
            assert bool(torch.isfinite(w).all())


@pytest.mark.parametrize("E,groups,keep,k", [(64, 32, 16, 4), (60, 30, 15, 4), (256, 8, 4, 4), (256, 8, 4, 12), (512, 32, 5, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_group_scores_that_cancel(E, groups, keep, k, score):
    """Large biases of both signs: a group's score is the small difference of large keys, whose rounding decides."""
    x = make(20000, E, E + k)
    size = E // groups
    for B in (16.0, 100.0, 1000.0, 1e5, 1e30):
        b = torch.full((E,), -B, device="cuda")
        b[::size] = B
        b += (torch.randn(E, generator=gen(3), device="cuda") * 0.01)
        idx, _ = ops.route_experts(x, k, score=score, bias=b, n_groups=groups, top_groups=keep)
        assert torch.equal(idx.long(), ro.choose(x, k, score, b, groups, keep)), B
        b = torch.full((E,), -B, device="cuda")
        b[::size] = B
        idx, _ = ops.route_experts(x, k, score=score, bias=b, n_groups=groups, top_groups=keep)
        assert torch.equal(idx.long(), ro.choose(x, k, score, b, groups, keep)), B


@pytest.mark.parametrize("E,groups,keep", [(64, 32, 2), (64, 32, 5), (60, 30, 3), (64, 8, 4), (256, 8, 4), (512, 32, 3)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biases_of_the_lowest_and_largest_value(E, groups, keep, score):
    """The sum of two keys of +-3.4e38 leaves fp32, the order of the groups does not: a mask of the type's lowest
    value puts experts last, but leaves them to choose from."""
    x = make(60, E, E)
    x[:20, ::3] = -INF
    x[20:30, :E // 2] = -INF
    size = E // groups
    last, one, rest, top, mixed = (torch.zeros(E, device="cuda") for _ in range(5))
    last[:E - size] = LOWEST                      # all but the last group
    one[:] = LOWEST
    one[E - 1] = 0.0                              # all but one expert
    rest[size:] = LOWEST
    rest[E // 2] = -INF
    top[::size] = -LOWEST                         # the largest value
    top[1::size] = -LOWEST
    top[:size] = 0.0
    mixed[::2] = LOWEST
    mixed[1::4] = -LOWEST
    for bias in (last, one, rest, top, mixed):
        for k in (2, 6, 8, 9):
            idx, w = ops.route_experts(x, k, score=score, bias=bias, n_groups=groups, top_groups=keep)
            assert torch.equal(idx.long(), ro.choose(x, k, score, bias, groups, keep))
            assert bool(torch.isfinite(w).all())


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("E,k", [(16, 3), (64, 6), (200, 8), (512, 32)])
def test_gradient_of_fp32_logits_far_from_the_maximum(score, renorm, E, k):
    """Experts up to 80 below the row's maximum keep fp32's relative accuracy. The logits are multiples of 2^-8, so
    their differences are exact and what is left is counted here in u = 2^-24: an exponential (2 ulps: 4), a sum of E
    terms (16 in a lane, 5 levels: 21, on top of the terms' 4), a reciprocal and products with it (1 each)."""
    n, u = 400, 2.0 ** -24
    g = gen(E)
    x = -torch.randint(0, 80 * 256, (n, E), generator=g, device="cuda").float() / 256
    x[:, 0] = 0.0
    idx = (torch.rand(n, E - 1, generator=g, device="cuda").argsort(1)[:, :k] + 1).int()
    dw = torch.randn(n, k, generator=g, device="cuda")
    d = ops.route_experts_backward(dw, x, idx, score=score, renormalize=renorm)
    l = x.double()
    at = idx.long()
    G = torch.zeros_like(l).scatter_(1, at, dw.double())
    if renorm:
        log = l if score == "softmax" else torch.nn.functional.logsigmoid(l)
        s = torch.softmax(torch.full_like(l, -INF).scatter(1, at, log.gather(1, at)), 1)
    else:
        s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    rest = torch.sigmoid(-l) if score == "sigmoid" else torch.ones_like(l)
    if score == "sigmoid" and not renorm:
        ref, A = s * rest * G, torch.zeros_like(l[:, :1])
        diff = G
    else:
        diff = G - (s * G).sum(1, keepdim=True)
        if renorm:
            diff = torch.zeros_like(l).scatter_(1, at, diff.gather(1, at))
        ref, A = s * rest * diff, (s * G.abs()).sum(1, keepdim=True)
    # s: 4 + 25 + 1 + 1; the inner sum: a product, 21 for its adds, 4, and the 25 + 2 of the division; G: the scale; the
    # last subtraction and two products. sigmoid: 1 + z, its reciprocal (1 ulp: 2) and a product in s, and in 1 - s, with z
    more = 6 + 10 if score == "sigmoid" else 0
    tol = u * s * rest * ((31 + 3 + more) * diff.abs() + (53 + more) * A + G.abs()) + 2.0 ** -126
    assert bool(((d.double() - ref).abs() <= tol).all()), float(((d.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("score,mul,off", [("softmax", 10.0, 0.0), ("sigmoid", 1.0, -20.0)])
def test_confident_rows_with_groups(score, mul, off):
    """Scores below fp32's error beside 1: the choice is the definition's, and takes no path of one token at a time."""
    x = make(65536, 256, 5)
    few = x[:3000] * mul + off
    for E, groups, keep, k in ((256, 8, 4, 8), (64, 8, 4, 4), (60, 3, 2, 8)):
        idx, _ = ops.route_experts(few[:, :E].contiguous(), k, score=score, n_groups=groups, top_groups=keep)
        assert torch.equal(idx.long(), ro.choose(few[:, :E], k, score, None, groups, keep))

    def time(t):
        best = INF
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.route_experts(t, 8, score=score, n_groups=8, top_groups=4)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(x * mul + off) < 8 * time(x)          # 2.5 times, where it was 22 and 48


@pytest.mark.parametrize("E,k", [(30, 4), (72, 15), (300, 9), (512, 32), (64, 8), (256, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_keys_at_the_border_hide_no_larger_one(E, k, score):
    """More equal experts than slots, and one after them that is larger by less than fp32 can tell."""
    x = torch.full((50, E), -9984.0, device="cuda")
    first = torch.arange(k // 2, device="cuda")
    x[:, first] = make(50, k // 2, E) + 2
    late = E - 1 - torch.arange(50, device="cuda") % (E // 4)
    x[torch.arange(50), late] = -20.0
    x[25:, E // 2] = -21.0
    for b in (torch.ones(E, device="cuda"), torch.zeros(E, device="cuda"), torch.full((E,), -3.0, device="cuda")):
        for t in (x, x.bfloat16()):
            idx, _ = ops.route_experts(t, k, score=score, bias=b)
            ref = ro.choose(t, k, score, b)
            assert torch.equal(idx.long(), ref)
            assert bool((ref == late[:, None]).any(1).all())
