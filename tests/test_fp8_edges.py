"""Shapes and strides of the general router's and the 8-bit operators that need no GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from agillm41_b200 import MoEKernelError, ops


def test_traced_experts_of_a_strided_batch_are_contiguous():
    """What a traced model is told about the output is what the kernels return, whatever the input's strides."""
    f8, u8 = torch.float8_e4m3fn, torch.uint8
    o = torch.ops.agillm_moe
    with FakeTensorMode():
        x = torch.empty(528, 300, dtype=torch.bfloat16, device="cuda").t()
        idx, w = torch.empty(300, 2, dtype=torch.int32, device="cuda"), torch.empty(300, 2, device="cuda")
        q1, q2 = torch.empty(8, 400, 528, dtype=f8, device="cuda"), torch.empty(8, 528, 400, dtype=f8, device="cuda")
        s1, s2 = torch.empty(8, 4, 2, 512, dtype=u8, device="cuda"), torch.empty(8, 5, 1, 512, dtype=u8, device="cuda")
        b1, b2 = torch.empty(8, 400, device="cuda"), torch.empty(8, 528, device="cuda")
        y = o.moe_experts_fp8(x, idx, w, q1, s1, b1, q2, s2, b2, None)
        assert y.shape == x.shape and y.is_contiguous()
        wide = [torch.empty(s, dtype=x.dtype, device="cuda") for s in ((8, 528), (8, 400, 528), (8, 400), (8, 528, 400), (8, 528))]
        assert o.moe_forward(x, *wide, 2).is_contiguous()


def test_sizes_past_the_c_ints_are_refused():
    """Widths, expert counts and k go through the C interface as 32-bit ints: larger ones are refused, not cut off."""
    big, bf16, f8, u8 = 2 ** 32, torch.bfloat16, torch.float8_e4m3fn, torch.uint8
    with FakeTensorMode():
        def t(*shape, dtype=bf16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        def fp8(*shape):
            tiles = ((shape[-2] + 127) // 128, (shape[-1] + 511) // 512, 512)
            return ops.FP8Tensor(t(*shape, dtype=f8), t(*shape[:-2], *tiles, dtype=u8))

        idx, w = t(4, 2, dtype=torch.int32), t(4, 2, dtype=torch.float32)
        calls = [lambda: ops.route_experts(t(1, big + 16), 2),
                 lambda: ops.route_experts(t(4, 16), big + 2),
                 lambda: ops.route_experts(t(4, 16), 2, n_groups=big + 1),
                 lambda: ops.route_experts(t(4, 16), 2, n_groups=4, top_groups=big + 1),
                 lambda: ops.route_experts(t(4, 16), 2 - big),
                 lambda: ops.route_experts_backward(t(1, big + 2, dtype=torch.float32), t(1, 16), t(1, big + 2, dtype=torch.int32)),
                 lambda: ops.quantize_fp8(t(1, big + 16)),
                 lambda: ops.quantize_fp8_weight(t(1, 16, big + 16)),
                 lambda: ops.quantize_fp8_weight(t(1, big + 16, 16)),
                 lambda: ops.dequantize_fp8(fp8(1, big + 16)),
                 lambda: ops.grouped_gemm_fp8(fp8(1, big + 16), fp8(1, 16, big + 16)),
                 lambda: ops.grouped_gemm_fp8(fp8(1, 16), fp8(1, big + 16, 16)),
                 lambda: ops.moe_experts_fp8(t(4, 16), idx, w, fp8(3, big + 16, 16), None, fp8(3, 16, big + 16), None),
                 lambda: ops.moe_experts_fp8(t(1, 16), t(1, big + 2, dtype=torch.int32), t(1, big + 2, dtype=torch.float32),
                                             fp8(3, 16, 16), t(3, 16, dtype=torch.float32), fp8(3, 16, 16),
                                             t(3, 16, dtype=torch.float32))]
        for i, call in enumerate(calls):
            with pytest.raises(MoEKernelError):
                call()
                pytest.fail(f"call {i} went through")
