"""General expert routing on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

from agillm41_b200 import MoEKernelError, ops, route_experts
from oracle import route_oracle as ro

pytestmark = pytest.mark.gpu

INF = math.inf
# Half a step of a rounding: relative in the normal range, absolute below it. fp16's normal range ends at 2^-14,
# below which its step is 2^-24; the other two end at 2^-126.
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(n, E, dtype=torch.float32, seed=0):
    return (torch.randn(n, E, generator=gen(seed), device="cuda") * 1.5).to(dtype)


def weight_bound(ref, E, k):
    """fp32 weights: an exponential within 2 ulps of its (rounded) argument, sums of at most E + k terms in a
    tree, a division and the scale: under 16 + log2(E) roundings, the argument's counted by its size (below 32
    for the logits here) as 32 more."""
    return (48 + math.log2(E) + k) * 2.0 ** -24 * ref.abs() + 1e-37


def check(logits, k, **kw):
    idx, w = ops.route_experts(logits, k, **kw)
    ck = {a: kw[a] for a in ("score", "bias", "n_groups", "top_groups") if a in kw}
    wk = {a: kw[a] for a in ("score", "renormalize", "scale") if a in kw}
    ref = ro.choose(logits, k, **ck)
    assert torch.equal(idx.long(), ref)
    rw = ro.weights(logits, ref, **wk)
    assert bool(((w.double() - rw).abs() <= weight_bound(rw, logits.shape[1], k)).all())
    return idx, w


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,E,k", [(1, 1, 1), (1, 14, 2), (9, 16, 16), (130, 17, 3), (64, 64, 8), (33, 65, 32), (257, 128, 6),
                                   (1000, 160, 6), (100, 256, 8), (31, 384, 8), (77, 512, 32)])
def test_plain(n, E, k, dtype, score):
    x = make(n, E, dtype, n + E)
    for renorm in (True, False):
        check(x, k, score=score, renormalize=renorm, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,E,k,groups,keep", [(50, 8, 2, 4, 2), (300, 256, 8, 8, 4), (65, 160, 6, 8, 3), (40, 32, 4, 32, 5),
                                               (200, 512, 8, 16, 1), (20, 60, 4, 3, 3), (20, 12, 3, 6, 2), (9, 48, 8, 2, 1)])
def test_groups_and_bias(n, E, k, groups, keep, dtype, score):
    x = make(n, E, dtype, n + E)
    b = torch.randn(E, generator=gen(E), device="cuda") * 0.1
    check(x, k, score=score, n_groups=groups, top_groups=keep)
    check(x, k, score=score, n_groups=groups, top_groups=keep, bias=b, renormalize=False)
    check(x, k, score=score, bias=b)
    check(x, k, score=score, bias=torch.zeros_like(b), n_groups=groups, top_groups=keep)


@pytest.mark.parametrize("E", [32, 33, 48, 61, 64, 90, 96, 128, 130, 160, 200, 252, 256, 260, 384, 509, 512])
def test_widths(E):
    """Expert counts that do and do not divide among lanes, with aligned and unaligned rows, for k on both sides of 8."""
    for dtype in (torch.float32, torch.bfloat16):
        x = make(67, E, dtype, E)
        b = torch.randn(E, generator=gen(E), device="cuda") * 0.1
        for k in (1, 5, 8, 9):
            check(x, k, score="sigmoid", bias=b)
            check(x, k, score="softmax", renormalize=False)
        for groups in (2, 4, 8, 16, 32):
            if E % groups == 0:
                for keep in {1, groups // 2}:
                    k = min(8, E // groups)
                    check(x, k, score="sigmoid", bias=b, n_groups=groups, top_groups=keep)
                    check(x, k, score="softmax", n_groups=groups, top_groups=keep)
        y = torch.empty(67 * E + 1, dtype=dtype, device="cuda")[1:].view(67, E).copy_(x)   # rows off their 16 bytes
        check(y, 6, score="sigmoid", bias=b)
        idx, w = ops.route_experts(y, 6)
        assert torch.equal(ops.route_experts_backward(w, y, idx), ops.route_experts_backward(w, x, idx))


def test_crowded_rows():
    """Rows where many keys tie or nearly tie at the border, up to all of them."""
    for E in (32, 64, 160, 256, 512):
        x = torch.zeros(40, E, device="cuda")
        x[:20] = torch.randint(0, 3, (20, E), generator=gen(E), device="cuda").float()
        x[30:] = make(10, E, seed=E) * 1e-7
        b = torch.randint(0, 2, (E,), generator=gen(1), device="cuda").float() * 0.25
        for bias in (None, b, b + torch.arange(E, device="cuda") * 2.0 ** -24):
            for score in ("softmax", "sigmoid"):
                check(x, 8, score=score, bias=bias)
                check(x, 8, score=score, bias=bias, n_groups=4, top_groups=2)


def test_many_tokens():
    """Enough near ties that some need the second look in 64 bits."""
    for dtype in (torch.float32, torch.bfloat16):
        x = make(40000, 256, dtype, 3)
        b = torch.randn(256, generator=gen(4), device="cuda") * 0.05
        check(x, 8, score="sigmoid", bias=b, n_groups=8, top_groups=4)
        check(x, 8, score="softmax", bias=b * 0.02)
        check(x, 6, score="softmax", n_groups=16, top_groups=3, renormalize=False)


@pytest.mark.parametrize("kw", [dict(top_k=8, score="sigmoid", n_groups=8, top_groups=4), dict(top_k=12), dict(top_k=6)])
def test_offsets_past_32_bits(kw):
    """More than 2^31 logits: the last rows come out as they do on their own."""
    x = torch.empty(9_000_003, 256, dtype=torch.bfloat16, device="cuda").normal_(generator=gen(5))
    last = x[-5000:].contiguous()
    score = kw.get("score", "softmax")
    idx, w = ops.route_experts(x, **kw)
    idx2, w2 = ops.route_experts(last, **kw)
    assert torch.equal(idx[-5000:], idx2) and torch.equal(w[-5000:], w2)
    d = ops.route_experts_backward(w, x, idx, score=score)
    assert torch.equal(d[-5000:], ops.route_experts_backward(w2, last, idx2, score=score))


def test_ties_go_to_the_lowest_index():
    x = torch.zeros(5, 48, device="cuda")
    x[1, 7] = x[1, 30] = x[1, 44] = 2.0
    x[2] = -0.0
    x[2, ::2] = 0.0
    x[3, 40:] = 1.0
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(48, device="cuda")):
            idx, _ = check(x, 5, score=score, bias=bias)
            assert idx[0].tolist() == [0, 1, 2, 3, 4] and idx[1].tolist() == [7, 30, 44, 0, 1]
            assert idx[2].tolist() == [0, 1, 2, 3, 4]
            check(x, 5, score=score, bias=bias, n_groups=6, top_groups=2)


def test_close_keys_are_told_apart():
    """Keys 2^-24 and less apart through score + bias: the order is that of the real numbers."""
    E, n = 64, 4096
    x = make(n, E, seed=8)
    target = 0.75 + torch.arange(E, device="cuda", dtype=torch.float64)[None, :] * 2.0 ** -26
    x64 = x.double()
    # a bias per expert cannot follow every token: use one token's scores, then copies with logits nudged by an ulp
    bias = (target - torch.sigmoid(x64[:1])).float().flatten()
    rows = x[:1].repeat(n, 1)
    nudge = torch.randint(-1, 2, (n, E), generator=gen(1), device="cuda", dtype=torch.int32)
    rows = (rows.view(torch.int32) + nudge).view(torch.float32)
    check(rows, 8, score="sigmoid", bias=bias)
    check(rows, 8, score="sigmoid", bias=bias, n_groups=8, top_groups=3)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,kw", [(14, {}), (40, {}), (200, {}), (64, dict(n_groups=8, top_groups=2))])
def test_masked_experts(score, E, kw):
    x = make(6, E, seed=E)
    x[0] = -INF                               # nothing left
    x[1, 1:] = -INF                           # one left
    x[2, ::2] = -INF
    x[3] = torch.finfo(torch.float32).min     # a mask of the type's lowest value leaves equal experts
    x[4, 3:] = torch.finfo(torch.float32).min
    for bias in (None, torch.linspace(-0.2, 0.2, E, device="cuda")):
        for renorm in (True, False):
            idx, w = check(x, 4, score=score, bias=bias, renormalize=renorm, **kw)
            assert idx[0].tolist() == [-1] * 4 and w[0].tolist() == [0.0] * 4
            assert idx[1].tolist() == [0, -1, -1, -1]
    off = torch.zeros(E, device="cuda")
    off[:5] = -INF                            # a bias takes experts out as well
    off[5] = float("nan")
    idx, _ = check(x[2:3], 4, score=score, bias=off, **kw)
    assert int(idx.min()) >= 6


def test_extreme_logits():
    """Renormalised weights do not underflow with their scores; large logits saturate."""
    x = torch.tensor([[-300.0, -301.0, -302.0, -1000.0], [90.0, 100.0, 110.0, 0.0], [-100.0, 50.0, -99.0, -98.0]], device="cuda")
    for score in ("softmax", "sigmoid"):
        _, w = check(x, 3, score=score)
        assert bool(torch.isfinite(w).all()) and bool((w.sum(1) - 1).abs().max() < 1e-6)


def test_nan_and_inf_rows():
    for E in (14, 64, 256):
        x = make(4, E, seed=1)
        x[1, 3] = float("nan")
        x[2, 5] = INF
        for score in ("softmax", "sigmoid"):
            idx, w = ops.route_experts(x, 2, score=score)
            clean = [0, 3] if score == "softmax" else [0, 2, 3]
            assert torch.equal(torch.isnan(w).any(1).nonzero().flatten().cpu(),
                               torch.tensor([i for i in range(4) if i not in clean]))
            assert torch.equal(idx[clean].long(), ro.choose(x[clean], 2, score))
            assert not bool((idx[1] == 3).any()) and int(idx.max()) < E


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,E,k", [(1, 14, 2), (33, 16, 5), (50, 64, 6), (70, 100, 32), (129, 256, 8), (10, 512, 4)])
def test_gradient(n, E, k, dtype, score, renorm):
    x = make(n, E, dtype, n)
    if n > 20:
        x[3] = -INF
        x[4, 2:] = -INF
    idx, _ = ops.route_experts(x, k, score=score, renormalize=renorm, scale=1.5)
    g = torch.randn(n, k, generator=gen(2), device="cuda")
    d = ops.route_experts_backward(g, x, idx, score=score, renormalize=renorm, scale=1.5)
    rows = [i for i in range(n) if not (n > 20 and i in (3, 4))]
    leaf = x.double().requires_grad_(True)
    w = ro.weights(leaf[rows], idx[rows], score, renorm, 1.5)
    (w * g[rows].double()).sum().backward()
    ref = leaf.grad[rows]
    # Terms w |g| of which a gradient is a difference, each within the weights' relative bound, then the output's rounding.
    mag = (ro.weights(x[rows], idx[rows], score, renorm, 1.5) * g[rows].double().abs()).sum(1, keepdim=True)
    s = ro.scores(x[rows].double(), score)
    own = torch.zeros_like(s).scatter_add_(1, idx[rows].long(), g[rows].double().abs() * 1.5)
    tol = (64 + 2 * math.log2(E) + 2 * k) * 2.0 ** -24 * (mag * torch.maximum(s, own / (own + 1)) + own) + HALF[dtype] * ref.abs() + TINY[dtype]
    assert bool(((d[rows].double() - ref).abs() <= tol).all()), float(((d[rows].double() - ref).abs() / tol).max())
    if n > 20:
        assert not bool(d[3].any()) and not bool(d[4, 2:].any()) and bool(torch.isfinite(d[4]).all())


def test_gradient_against_differences():
    x = make(6, 24, seed=5)
    g = torch.randn(6, 4, generator=gen(6), device="cuda")
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            idx, _ = ops.route_experts(x, 4, score=score, renormalize=renorm)
            d = ops.route_experts_backward(g, x, idx, score=score, renormalize=renorm)
            h = 1e-4
            for e in range(0, 24, 5):
                up, down = x.double(), x.double()
                up[:, e] += h
                down[:, e] -= h
                diff = ((ro.weights(up, idx, score, renorm) - ro.weights(down, idx, score, renorm)) * g.double()).sum(1) / (2 * h)
                # central differences are off by h^2 / 6 times a third derivative (below 8 sum |g| here)
                assert bool(((d[:, e].double() - diff).abs() <= 8 * h * h * g.double().abs().sum(1) + 1e-6).all())


def test_gradient_repeated_and_empty_slots():
    x = make(3, 20, seed=7)
    idx = torch.tensor([[4, 4, 9], [-1, 2, -1], [25, -7, 19]], dtype=torch.int32, device="cuda")
    g = torch.randn(3, 3, generator=gen(8), device="cuda")
    d = ops.route_experts_backward(g, x, idx, score="sigmoid", renormalize=False)
    s = torch.sigmoid(x.double())
    ref = torch.zeros_like(s)
    for t in range(3):
        for r in range(3):
            e = int(idx[t, r])
            if 0 <= e < 20:
                ref[t, e] += g[t, r].double() * s[t, e] * (1 - s[t, e])
    torch.testing.assert_close(d.double(), ref, rtol=0, atol=64 * 2.0 ** -24 * float(g.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(dtype):
    """The differentiable form: weights carry the gradient, indices none; the bias gets none."""
    x = make(40, 32, dtype, 9).requires_grad_(True)
    b = torch.zeros(32, device="cuda", requires_grad=True)
    idx, w = route_experts(x, 4, score="sigmoid", bias=b, n_groups=4, top_groups=2, scale=2.0)
    g = torch.randn(40, 4, generator=gen(1), device="cuda")
    (w * g).sum().backward()
    assert not idx.requires_grad and b.grad is None
    assert torch.equal(x.grad, ops.route_experts_backward(g, x.detach(), idx, score="sigmoid", scale=2.0))
    with torch.no_grad():
        assert not route_experts(x, 4)[1].requires_grad


def test_autograd_once():
    """A second derivative is refused, not taken as zero."""
    x = make(5, 9).requires_grad_()
    _, w = route_experts(x, 2)
    g, = torch.autograd.grad(w.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_routing_then_experts():
    """A run of the operators together: router logits, grouped sigmoid routing with a balance bias, 8-bit experts,
    and the gradient back to the router."""
    n, d, H, E, k = 300, 256, 384, 32, 4
    x = torch.randn(n, d, generator=gen(1), device="cuda").to(torch.bfloat16)
    wr = (torch.randn(E, d, generator=gen(2), device="cuda") * d ** -0.5).requires_grad_(True)
    w1 = ops.quantize_fp8_weight(torch.randn(E, H, d, generator=gen(3), device="cuda") * d ** -0.5)
    w2 = ops.quantize_fp8_weight(torch.randn(E, d, H, generator=gen(4), device="cuda") * H ** -0.5)
    b1, b2 = torch.zeros(E, H, device="cuda"), torch.zeros(E, d, device="cuda")
    bias = torch.randn(E, generator=gen(5), device="cuda") * 0.1
    idx, w = route_experts(x.float() @ wr.t(), k, score="sigmoid", bias=bias, n_groups=8, top_groups=4, scale=2.5)
    y = ops.moe_experts_fp8(x, idx, w.detach(), w1, b1, w2, b2, residual=x, check_errors=True)
    # one expert at a time, by the slots that chose it, through the same products
    parts = torch.zeros(n, d, device="cuda", dtype=torch.float64)
    for r in range(k):
        one = torch.full_like(idx, -1)
        one[:, r] = idx[:, r]
        parts += ops.moe_experts_fp8(x, one, torch.ones_like(w), w1, b1, w2, b2).double() * w[:, r:r + 1].detach().double()
    ref = x.double() + parts
    assert bool(((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5).all())
    (w * torch.randn_like(w)).sum().backward()
    assert bool(torch.isfinite(wr.grad).all()) and float(wr.grad.abs().sum()) > 0


def test_capture_and_streams():
    x = make(500, 64, seed=3)
    ref = ops.route_experts(x, 6, score="sigmoid")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        idx, w = ops.route_experts(x, 6, score="sigmoid")
        d = ops.route_experts_backward(w, x, idx, score="sigmoid")
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(idx, ref[0]) and torch.equal(w, ref[1])
    assert torch.equal(d, ops.route_experts_backward(ref[1], x, ref[0], score="sigmoid"))


def test_no_tokens():
    idx, w = ops.route_experts(torch.empty(0, 8, device="cuda"), 2)
    assert idx.shape == (0, 2) and w.shape == (0, 2)
    assert ops.route_experts_backward(w, torch.empty(0, 8, device="cuda"), idx).shape == (0, 8)


def test_refusals():
    x = make(4, 16)
    for bad in (dict(top_k=17), dict(top_k=0), dict(top_k=2, score="tanh"), dict(top_k=2, n_groups=3),
                dict(top_k=2, n_groups=4, top_groups=5), dict(top_k=2, n_groups=4, top_groups=0),
                dict(top_k=2, bias=torch.zeros(15, device="cuda")), dict(top_k=2, bias=torch.zeros(16)),
                dict(top_k=2, bias=torch.zeros(16, device="cuda", dtype=torch.bfloat16))):
        k = bad.pop("top_k")
        with pytest.raises(MoEKernelError):
            ops.route_experts(x, k, **bad)
    with pytest.raises(MoEKernelError):
        ops.route_experts(make(4, 513), 2)
    with pytest.raises(MoEKernelError):
        ops.route_experts(make(4, 64), 33)
    with pytest.raises(MoEKernelError):
        ops.route_experts(x.t(), 2)
    with pytest.raises(MoEKernelError):
        ops.route_experts(x.double(), 2)
    with pytest.raises(MoEKernelError):
        ops.route_experts(x[0], 2)
    idx, w = ops.route_experts(x, 2)
    with pytest.raises(MoEKernelError):
        ops.route_experts_backward(w, x, idx.long())
    with pytest.raises(MoEKernelError):
        ops.route_experts_backward(w[:2], x, idx)
    with pytest.raises(MoEKernelError):
        ops.route_experts_backward(w.bfloat16(), x, idx)
