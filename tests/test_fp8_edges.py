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
