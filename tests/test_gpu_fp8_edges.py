"""Block-scaled e4m3 at the ends of the types' ranges, and what a call leaves as it was."""
import pytest
import torch

from agillm41_b200 import ops
from oracle import fp8_oracle as fo

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_largest_values_round_up_past_the_range(dtype):
    """The largest value of each type is nearer to the power of two above it than to the e4m3 value below: it stands for
    that power, which its own type does not have, and a larger type does."""
    top = torch.finfo(dtype).max
    x = torch.zeros(2, 128, dtype=dtype, device="cuda")
    x[0, 0], x[0, 1] = top, -top
    # 15/16 of the power of two is an e4m3 value
    x[1, 0] = torch.tensor(2.0 ** {torch.float16: 16}.get(dtype, 128) * 15 / 16, dtype=torch.float64).to(dtype)
    t = ops.quantize_fp8(x)
    q, p = fo.quantize(x.double())
    assert torch.equal(t.q.float().double(), q) and torch.equal(t.scales.cpu(), fo.tiles_of(p))
    stands = fo.values(q, p)
    assert float(stands[0, 0]) == 2.0 ** (16 if dtype == torch.float16 else 128)
    got = ops.dequantize_fp8(t, dtype)
    assert float(got[0, 0]) == float("inf") and float(got[0, 1]) == -float("inf") and torch.equal(got[1], x[1])
    if dtype == torch.float16:
        assert torch.equal(ops.dequantize_fp8(t, torch.float32).double(), stands)


@pytest.mark.parametrize("rows,width", [(1, 16), (130, 144), (1000, 1296)])
def test_weights_end_where_their_tensor_ends(rows, width):
    """Nothing is written behind the last row of weights."""
    x = torch.randn(rows, width, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda")
    pad = torch.full((rows + 300, width), 5, dtype=torch.uint8, device="cuda")
    w = ops.FP8Tensor(pad[:rows].view(torch.float8_e4m3fn)[None], torch.empty(1, -(-rows // 128), -(-width // 512), 512,
                                                                                dtype=torch.uint8, device="cuda"))
    ops.quantize_fp8_weight(x[None], out=w)
    assert bool((pad[rows:] == 5).all())
    q, p = fo.quantize(x.double(), 128)
    assert torch.equal(w.q[0].float().double(), q)


def test_e4m3_products_into_a_given_tensor():
    """Rows of no segment keep their bytes, under scale bytes of 0."""
    g = torch.Generator(device="cuda").manual_seed(1)
    a = ops.quantize_fp8(torch.randn(512, 128, generator=g, device="cuda"))
    w = ops.quantize_fp8_weight(torch.randn(2, 144, 128, generator=g, device="cuda"))
    seg = torch.tensor([0, 256, 384], dtype=torch.int32, device="cuda")
    cnt = torch.tensor([100, 128], dtype=torch.int32, device="cuda")
    out = torch.full((512, 144), 5, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    y = ops.grouped_gemm_fp8(a, w, seg_start=seg, counts=cnt, out_dtype=torch.float8_e4m3fn, out=out)
    assert y.q.data_ptr() == out.data_ptr()
    raw = out.view(torch.uint8)
    assert bool((raw[128:256] == 5).all()) and bool((raw[384:] == 5).all()) and not bool(raw[100:128].any())
    assert not bool(y.scales[1].any()) and not bool(y.scales[3].any()) and bool(y.scales[2].any())


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_products_without_rows(out_dtype):
    w = ops.quantize_fp8_weight(torch.randn(2, 32, 64, device="cuda"))
    a = ops.quantize_fp8(torch.empty(0, 64, device="cuda"))
    seg, cnt = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    y = ops.grouped_gemm_fp8(a, w, seg_start=seg, counts=cnt, out_dtype=out_dtype)
    one = ops.FP8Tensor(w.q[:1].contiguous(), w.scales[:1].contiguous())
    z = ops.grouped_gemm_fp8(a, one, out_dtype=out_dtype)
    for t in (y, z):
        if out_dtype == torch.float8_e4m3fn:
            assert t.q.shape == (0, 32) and t.scales.shape == (0, 1, 512)
            assert ops.dequantize_fp8(t).shape == (0, 32)
        else:
            assert t.shape == (0, 32)
    none = ops.quantize_fp8_weight(torch.empty(0, 32, 64, device="cuda"))
    assert none.q.shape == (0, 32, 64) and ops.dequantize_fp8(none).shape == (0, 32, 64)
