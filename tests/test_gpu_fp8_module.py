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
