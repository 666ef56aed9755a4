"""MoEFFN with 8-bit experts: device errors, sums, refusals."""
import pytest
import torch

import agillm41_b200
from agillm41_b200 import ops

pytestmark = pytest.mark.gpu

Error = agillm41_b200.MoEKernelError


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def module(d=256, experts=6, top_k=2, shared=1, dtype=torch.bfloat16, seed=3):
    torch.manual_seed(seed)
    m = agillm41_b200.MoEFFN(d, mlp_mult=2, experts=experts, top_k=top_k, shared_experts=shared, shared_mlp_mult=1)
    for blk in (m.shared or []):
        torch.nn.init.normal_(blk[2].weight, std=0.05)
        torch.nn.init.normal_(blk[2].bias, std=0.1)
    m = m.to(device="cuda", dtype=dtype).eval()
    m.expert_precision = "fp8"
    return m


@pytest.mark.parametrize("stage", ["router_topk", "grouped_gemm_fp8"])
def test_device_errors_of_every_stage_are_reported(stage, monkeypatch):
    """check_device_errors sees the router's and the shared experts' error words, as it sees the routed experts'."""
    m = module()
    x = torch.randn(70, 256, generator=gen(1), device="cuda").bfloat16()
    with torch.no_grad():
        ref = m(x)
        m.check_device_errors = True
        assert torch.equal(m(x), ref)
        real = getattr(ops, stage)

        def gives_up(*args, err=None, **kw):
            out = real(*args, err=err, **kw)
            if err is not None:
                err.fill_(4)                       # as a wait that ran out
            return out

        monkeypatch.setattr(ops, stage, gives_up)
        with pytest.raises(Error, match="0x4"):
            m(x)
        m.check_device_errors = False
        assert torch.equal(m(x), ref)


def expected(m, x, res):
    """The module's sum in 64 bits with what its parts may be off: each y by its rounding and its sums."""
    from oracle import fp8_oracle as fo
    n, d = x.shape
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[x.dtype]

    def part(mods, idx, w):
        q = [fo.read(ops.quantize_fp8_weight(torch.stack([ex[i].weight for ex in mods]))) for i in (0, 2)]
        b = [torch.stack([ex[i].bias for ex in mods]).float() for i in (0, 2)]
        return q[0], b[0], q[1], b[1]

    def rounded_sum(mods, idx, w):                  # value, and its bound without the rounding of the sum itself
        ref, tol = fo.experts(x.double(), idx, w, *part(mods, idx, w), half)
        return ref, (tol - half * ref.abs()) / (1 + half)

    idx, gates, _, _ = ops.router_topk(x, m.router.weight.contiguous(), m.top_k)
    ref, tol = rounded_sum(m.experts, idx, gates.float())
    for blk in (m.shared or []):
        # one expert of weight 1: its sum is y itself, which has one rounding
        y, t = fo.experts(x.double(), torch.zeros(n, 1, dtype=torch.int32, device="cuda"), torch.ones(n, 1, device="cuda"),
                          *part([blk], None, None), 0.0)
        ref, tol = ref + y, tol + t + half * (y.abs() + t)
    if res is not None:
        ref = ref + res.double()
    tol = tol + (m.top_k + 4) * 2.0 ** -24 * (ref.abs() + (0 if res is None else res.double().abs()) + 1)   # fp32 adds
    return ref, tol + half * (ref.abs() + tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared", [1, 3])
@pytest.mark.parametrize("n", [40, 1500])
def test_shared_experts_and_residual_are_summed_before_the_rounding(n, shared, dtype):
    """Residual, shared experts and routed experts are one fp32 sum with one rounding at its end."""
    m = module(shared=shared, dtype=dtype)
    x = torch.randn(n, 256, generator=gen(1), device="cuda").to(dtype)
    res = (torch.randn(n, 256, generator=gen(2), device="cuda") * 30).to(dtype)
    with torch.no_grad():
        got = m.forward_residual(x, res)
        ref, tol = expected(m, x, res)
        assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() / tol).max())
        ref, tol = expected(m, x, None)
        assert bool(((m(x).double() - ref).abs() <= tol).all())


def test_partial_sums_may_leave_fp16():
    """60000 + 20000 - 30000 is a fp16 number, 60000 + 20000 is none."""
    m = module(shared=1, dtype=torch.float16)
    with torch.no_grad():
        m.shared[0][2].bias.fill_(20000.0)
        for ex in m.experts:
            ex[2].bias.fill_(-30000.0)
        x = torch.randn(50, 256, generator=gen(1), device="cuda").half()
        res = torch.full_like(x, 60000.0)
        got = m.forward_residual(x, res)
        ref, tol = expected(m, x, res)
        assert bool(torch.isfinite(got).all()) and bool(((got.double() - ref).abs() <= tol).all())


def test_shared_outputs_are_checked():
    E, d, H, n = 3, 64, 128, 8
    x = torch.randn(n, d, generator=gen(1), device="cuda").bfloat16()
    w1 = ops.quantize_fp8_weight(torch.randn(E, H, d, generator=gen(2), device="cuda"))
    w2 = ops.quantize_fp8_weight(torch.randn(E, d, H, generator=gen(3), device="cuda"))
    b1, b2 = torch.zeros(E, H, device="cuda"), torch.zeros(E, d, device="cuda")
    idx, w = ops.route_experts(torch.randn(n, E, generator=gen(4), device="cuda"), 2)
    ref = ops.moe_experts_fp8(x, idx, w, w1, b1, w2, b2)
    none = torch.empty(0, n, d, dtype=x.dtype, device="cuda")
    assert torch.equal(ops.moe_experts_fp8(x, idx, w, w1, b1, w2, b2, shared=none), ref)
    for bad in (x, x[None].float(), x[None, :4], x[None].cpu(), torch.zeros(2, n, 2 * d, dtype=x.dtype, device="cuda")[:, :, ::2]):
        with pytest.raises(Error):
            ops.moe_experts_fp8(x, idx, w, w1, b1, w2, b2, shared=bad)


def test_gradients_of_the_residual_are_refused_too():
    """A frozen module and an input without gradient, but a residual with one: its gradient would be lost."""
    m = module().requires_grad_(False)
    x = torch.randn(20, 256, generator=gen(1), device="cuda").bfloat16()
    res = torch.randn_like(x)
    ref = m.forward_residual(x, res)
    with pytest.raises(Error, match="no_grad"):
        m.forward_residual(x, res.requires_grad_())
    with torch.no_grad():
        assert torch.equal(m.forward_residual(x, res), ref)


def test_parameters_made_in_inference_mode():
    """They have no version counter: quantised in every call, and a capture is refused with that reason."""
    with torch.inference_mode():
        m = module()
        x = torch.randn(20, 256, generator=gen(1), device="cuda").bfloat16()
        first = m(x)
        m.experts[0][0].weight.mul_(1.5)
        assert not torch.equal(m(x), first)
        with pytest.raises(Error, match="version counter"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                m(x)


def test_no_tokens_with_shared_experts():
    m = module()
    m.check_device_errors = True
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        assert m(x).shape == (0, 256) and m.forward_residual(x, x).shape == (0, 256)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("n,d", [(50, 272), (12000, 256), (2500, 1296)])
def test_shared_outputs_in_every_form_of_the_sum(n, d, k):
    """Few and many tokens, one and several parts of a row: shared outputs of zeros change nothing, and without routed
    rows the sum is the fp32 one of residual and shared outputs, rounded once."""
    E, H, dtype = 5, 128, torch.float16
    w1 = ops.quantize_fp8_weight(torch.randn(E, H, d, generator=gen(1), device="cuda") * d ** -0.5)
    w2 = ops.quantize_fp8_weight(torch.randn(E, d, H, generator=gen(2), device="cuda") * H ** -0.5)
    rest = (w1, torch.zeros(E, H, device="cuda"), w2, torch.ones(E, d, device="cuda"))
    x = torch.randn(n, d, generator=gen(3), device="cuda").to(dtype)
    idx = torch.randint(0, E, (n, k), generator=gen(4), device="cuda", dtype=torch.int32)
    w = torch.randn(n, k, generator=gen(5), device="cuda")
    sh = torch.randn(3, n, d, generator=gen(6), device="cuda").to(dtype) * 30
    plain = ops.moe_experts_fp8(x, idx, w, *rest, residual=x)
    assert torch.equal(ops.moe_experts_fp8(x, idx, w, *rest, residual=x, shared=torch.zeros_like(sh)), plain)
    assert not torch.equal(ops.moe_experts_fp8(x, idx, w, *rest, residual=x, shared=sh), plain)
    none = torch.full_like(idx, -1)
    got = ops.moe_experts_fp8(x, none, w, *rest, residual=x, shared=sh)
    assert torch.equal(got, (((x.float() + sh[0].float()) + sh[1].float()) + sh[2].float()).to(dtype))
    got = ops.moe_experts_fp8(x, none, w, *rest, shared=sh[:1].contiguous())
    assert torch.equal(got, sh[0])
