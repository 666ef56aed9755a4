"""Refusals and definitions of the general router and the 8-bit path that need no GPU."""
import ctypes
import math

import pytest
import torch

from agillm41_b200 import MoEKernelError, _lib, ops
from oracle import fp8_oracle as fo
from oracle import route_oracle as ro

FAKE = ctypes.c_void_p(4096)   # never read: the checks come first
ODD = ctypes.c_void_p(4096 + 8)


def message():
    return _lib.load().agm_last_error().decode()


@pytest.mark.parametrize("change,code", [
    (dict(dtype=9), -1), (dict(n=-1), -1), (dict(E=0), -2), (dict(E=513, k=2), -2), (dict(k=0), -1), (dict(k=65), -1),
    (dict(k=33), -2), (dict(score=2), -1), (dict(groups=5), -1), (dict(groups=0), -1), (dict(groups=64, top=1), -1),
    (dict(groups=8, top=9), -1), (dict(groups=8, top=0), -1), (dict(logits=None), -1), (dict(idx=None), -1),
    (dict(weights=None), -1)])
def test_route_arguments(change, code):
    a = dict(logits=FAKE, dtype=_lib.AGM_F32, n=8, E=64, k=4, score=0, bias=None, groups=1, top=1, idx=FAKE, weights=FAKE)
    a.update(change)
    rc = _lib.load().agm_route_experts(a["logits"], a["dtype"], a["n"], a["E"], a["k"], a["score"], a["bias"], a["groups"],
                                       a["top"], 1, 1.0, a["idx"], a["weights"], None)
    assert rc == code and message()


def test_route_backward_arguments():
    lib = _lib.load()
    assert lib.agm_route_experts_backward(FAKE, FAKE, 0, 8, 64, 33, FAKE, 0, 1, 1.0, FAKE, None) == -2
    assert lib.agm_route_experts_backward(FAKE, FAKE, 0, 8, 64, 4, None, 0, 1, 1.0, FAKE, None) == -1
    assert lib.agm_route_experts_backward(FAKE, FAKE, 0, 0, 64, 4, FAKE, 0, 1, 1.0, FAKE, None) == 0


def test_fp8_sizes_and_arguments():
    lib = _lib.load()
    assert lib.agm_fp8_scale_bytes(1, 16) == 512 and lib.agm_fp8_scale_bytes(129, 513) == 4 * 512
    assert lib.agm_fp8_scale_bytes(0, 16) == 0
    assert lib.agm_quantize_fp8(FAKE, 7, 8, 64, FAKE, FAKE, None) == -1
    assert lib.agm_quantize_fp8(FAKE, 0, 8, 24, FAKE, FAKE, None) == -2
    assert lib.agm_quantize_fp8(FAKE, 0, -1, 64, FAKE, FAKE, None) == -1
    assert lib.agm_quantize_fp8(ODD, 0, 8, 64, FAKE, FAKE, None) == -1
    assert lib.agm_quantize_fp8(FAKE, 0, 0, 64, FAKE, FAKE, None) == 0
    assert lib.agm_quantize_fp8_weight(FAKE, 0, 70000, 64, 64, FAKE, FAKE, None) == -2
    assert lib.agm_quantize_fp8_weight(FAKE, 0, 2, 64, 60, FAKE, FAKE, None) == -2
    assert lib.agm_dequantize_fp8(FAKE, FAKE, 1, 8, 64, 5, FAKE, None) == -1
    assert lib.agm_dequantize_fp8(FAKE, None, 1, 8, 64, 0, FAKE, None) == -1


@pytest.mark.parametrize("change,code", [
    (dict(groups=513, seg=FAKE, cnt=FAKE), -2), (dict(groups=2), -1), (dict(seg=FAKE), -1), (dict(n=24), -2), (dict(k=8), -2),
    (dict(c_dtype=0), -1), (dict(mode=3), -1), (dict(a=None), -1), (dict(c=ODD), -1), (dict(bias=ODD), -1), (dict(rows=-1), -1),
    (dict(rows=2 ** 31), -2)])
def test_product_arguments(change, code):
    a = dict(a=FAKE, rows=128, bias=None, groups=1, n=64, k=64, seg=None, cnt=None, mode=0, c=FAKE, c_dtype=_lib.AGM_BF16)
    a.update(change)
    rc = _lib.load().agm_grouped_gemm_fp8(a["a"], FAKE, a["rows"], FAKE, FAKE, a["bias"], a["groups"], a["n"], a["k"], a["seg"],
                                          a["cnt"], 0, a["mode"], a["c"], a["c_dtype"], None, None, None)
    assert rc == code and message()


def test_experts_arguments():
    lib = _lib.load()
    n, d, E, k, H = 64, 128, 14, 2, 256
    need = lib.agm_moe_experts_fp8_workspace_bytes(n, d, E, k, H)
    rows = -(-(n * k + E * 127) // 128) * 128
    assert need >= rows * (d + H + 2 * d)
    assert lib.agm_moe_experts_fp8_workspace_bytes(1, d, 512, 2, H) < lib.agm_moe_experts_fp8_workspace_bytes(9, d, 512, 2, H)

    def call(dtype=_lib.AGM_BF16, n=n, d=d, E=E, k=k, H=H, w1=FAKE, out=FAKE, ws=FAKE, ws_bytes=1 << 40):
        return lib.agm_moe_experts_fp8(FAKE, dtype, n, d, E, k, H, FAKE, FAKE, w1, FAKE, FAKE, FAKE, FAKE, FAKE, None, out,
                                       ws, ws_bytes, None)

    assert call(dtype=_lib.AGM_F32) == -2
    assert call(d=24) == -2 and call(H=100) == -2 and call(E=513) == -2
    assert call(k=0) == -1 and call(k=33) == -1 and call(n=-1) == -1
    assert call(w1=None) == -1 and call(out=ODD) == -1 and call(ws=None) == -1
    assert call(ws_bytes=need - 1) == -5 and "workspace" in message()
    assert call(n=2 ** 31) == -2


def test_cpu_tensors_are_refused():
    x = torch.zeros(8, 64)
    t = ops.FP8Tensor(torch.zeros(8, 64, dtype=torch.float8_e4m3fn), torch.zeros(1, 1, 512, dtype=torch.uint8))
    for call in (lambda: ops.route_experts(x, 2), lambda: ops.quantize_fp8(x), lambda: ops.quantize_fp8_weight(x[None]),
                 lambda: ops.dequantize_fp8(t), lambda: ops.grouped_gemm_fp8(t, t),
                 lambda: ops.route_experts_backward(x, x, x.int())):
        with pytest.raises(MoEKernelError):
            call()


def test_oracle_rounding_is_torchs():
    """The oracle's e4m3 rounding against torch's cast, over all neighbours and midpoints of the type."""
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    v = v[torch.isfinite(v)].unique()
    mid = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    assert torch.equal(fo.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_oracle_scales_and_tiles():
    amax = torch.tensor([448.0, 448.0001, 0.0, 1.0, 1.75, 1.7500001, 2.0 ** -140], dtype=torch.float64)
    p = fo.exponent(amax)
    assert p.tolist() == [0, 1, -127, -8, -8, -7, -127]
    e = torch.randint(-100, 100, (300, 7)).double()
    assert torch.equal(fo.exponents_of(fo.tiles_of(e), 300, 7), e)


def test_oracle_routing_by_hand():
    l = torch.tensor([[0.0, 3.0, 1.0, 2.0, -1.0, 2.5]])
    assert ro.choose(l, 3).tolist() == [[1, 5, 3]]
    # three groups of two: sums (sigmoid) .5+.95, .73+.88, .27+.92
    assert ro.choose(l, 3, "sigmoid", None, 3, 1).tolist() == [[3, 2, -1]]
    bias = torch.tensor([9.0, 0.0, 0.0, 0.0, 9.0, 0.0])
    assert ro.choose(l, 2, "sigmoid", bias).tolist() == [[0, 4]]
    assert ro.choose(torch.full((1, 4), -math.inf), 2).tolist() == [[-1, -1]]
    w = ro.weights(l, torch.tensor([[1, 5, -1]]), "softmax", True, 2.0)
    assert torch.allclose(w, torch.tensor([[2 / (1 + math.exp(-0.5)), 2 / (1 + math.exp(0.5)), 0.0]], dtype=torch.float64))


def test_torch_operators_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    f8 = torch.float8_e4m3fn
    o = torch.ops.agillm_moe
    with FakeTensorMode():
        x = torch.empty(300, 528, dtype=torch.bfloat16, device="cuda")
        idx, w = o.route_experts(torch.empty(300, 64, device="cuda"), 6, "sigmoid", None, 8, 4, True, 2.5)
        assert idx.shape == w.shape == (300, 6) and idx.dtype == torch.int32 and w.dtype == torch.float32
        q, s = o.quantize_fp8(x)
        assert q.shape == x.shape and q.dtype == f8 and s.shape == (3, 2, 512) and s.dtype == torch.uint8
        assert o.dequantize_fp8(q, s, torch.float32).dtype == torch.float32
        w1, s1 = o.quantize_fp8_weight(torch.empty(64, 400, 528, device="cuda"))
        w2, s2 = o.quantize_fp8_weight(torch.empty(64, 528, 400, device="cuda"))
        assert s1.shape == (64, 4, 2, 512) and s2.shape == (64, 5, 1, 512)
        y = o.grouped_gemm_fp8(q, s, w1, s1, None, True, idx[:65, 0], idx[:64, 0], torch.float16)
        assert y.shape == (300, 400) and y.dtype == torch.float16
        b1, b2 = torch.empty(64, 400, device="cuda"), torch.empty(64, 528, device="cuda")
        assert o.moe_experts_fp8(x, idx, w, w1, s1, b1, w2, s2, b2, None).shape == x.shape


def test_module_precision_is_checked():
    import agillm41_b200

    m = agillm41_b200.MoEFFN(64, mlp_mult=2, experts=4, top_k=2)
    assert m.expert_precision == "model"
    m.expert_precision = "fp8"
    with pytest.raises(MoEKernelError):
        m(torch.zeros(3, 64))                    # no CPU path
    with pytest.raises(MoEKernelError):
        with torch.no_grad():
            m.forward_host(torch.zeros(3, 64))
