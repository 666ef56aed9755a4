"""Block-scaled e4m3 on the GPU against its definition in 64 bits: quantisation
and its inverse bit for bit, the grouped products and the experts' forward to
bounds counted from their roundings."""
import copy
import io

import pytest
import torch

import agillm41_b200
from agillm41_b200 import _lib, ops
from oracle import fp8_oracle as fo

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
ROWS, WEIGHTS = _lib.AGM_FP8_ROWS, _lib.AGM_FP8_WEIGHTS


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def acts(rows, width, seed, dtype=torch.float32, spread=0.5):
    g = gen(seed)
    x = torch.randn(rows, width, generator=g, device="cuda")
    return (x * torch.exp(spread * torch.randn(width, generator=g, device="cuda"))).to(dtype)


def weight(G, n, width, seed, dtype=torch.float32):
    return (torch.randn(G, n, width, generator=gen(seed), device="cuda") * width ** -0.5).to(dtype)


# ---------------------------------------------------------------------------
# Quantisation
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(1, 16), (1, 128), (3, 144), (127, 512), (128, 528), (129, 1280), (1000, 2000)])
def test_quantize_rows(rows, width, dtype):
    x = acts(rows, width, rows + width, dtype, spread=2.0)
    t = ops.quantize_fp8(x)
    q, p = fo.quantize(x.double())
    assert torch.equal(t.q.float().double(), q)
    assert torch.equal(t.scales.cpu(), fo.tiles_of(p))
    for out in (torch.float32, torch.bfloat16, torch.float16):
        # The values are exact in fp64; torch's cast rounds once, to nearest even. (An e4m3 value times a power
        # of two is exact in fp32, so fp64 -> fp32 -> 16 bits is one rounding too.)
        assert torch.equal(ops.dequantize_fp8(t, out), fo.values(q, p).float().to(out))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,n,width", [(1, 16, 16), (2, 128, 128), (3, 144, 272), (2, 400, 1280), (5, 130, 640)])
def test_quantize_weight(G, n, width, dtype):
    w = weight(G, n, width, n + width, dtype) * torch.exp2(torch.arange(G, device="cuda") * 3.0)[:, None, None].to(dtype)
    t = ops.quantize_fp8_weight(w)
    q, p = fo.quantize(w.double(), 128)
    assert torch.equal(t.q.float().double(), q)
    rows = fo.row_exponents(p, -(-n // 128) * 128, 128)
    for g in range(G):
        assert torch.equal(t.scales[g].cpu(), fo.tiles_of(rows[g]))
    assert torch.equal(ops.dequantize_fp8(t, torch.float32).double(), fo.values(q, rows[:, :n]))


def test_quantize_borders():
    """Maxima at and next to 448 * 2^p, ties between e4m3 values, subnormals, zeros, the ends of fp32's range."""
    rows = []
    for top in (448.0, 449.0, 447.0, 480.0, 240.0, 1.75, 1.76, 2.0 ** -126, 2.0 ** -130, 2.0 ** -149, 0.0, 3.4e38, 1.0e-30):
        r = torch.linspace(-1, 1, 128, dtype=torch.float64) * top
        r[0] = top
        rows.append(r)
    ties = torch.arange(128, dtype=torch.float64) / 8 + 1.0 / 16      # between neighbours of the first octaves
    ties[127] = 448
    rows.append(ties)
    tiny = torch.arange(128, dtype=torch.float64) * 2.0 ** -10         # halves of the subnormal step
    tiny[127] = 448
    rows.append(tiny)
    x = torch.stack(rows).float().cuda()
    t = ops.quantize_fp8(x)
    q, p = fo.quantize(x.double())
    assert torch.equal(t.q.float().double(), q)
    assert torch.equal(t.scales.cpu(), fo.tiles_of(p))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_quantize_non_finite_stays_visible_and_alone(bad):
    x = acts(4, 256, 1)
    x[1, 3] = bad
    x[2, 128:] = bad
    t = ops.quantize_fp8(x)
    q, p = fo.quantize(x.double())
    got = ops.dequantize_fp8(t, torch.float32)
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x))
    torch.testing.assert_close(got.double(), fo.values(q, p), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_weight_non_finite(dtype):
    w = weight(2, 200, 272, 3, dtype)
    w[0, 5, 7], w[0, 130, 200], w[1, 199, 271] = float("inf"), float("nan"), -float("inf")
    t = ops.quantize_fp8_weight(w)
    q, p = fo.quantize(w.double(), 128)
    got = ops.dequantize_fp8(t, torch.float32)
    assert int(torch.isnan(got).sum()) == 3
    torch.testing.assert_close(got.double(), fo.values(q, fo.row_exponents(p, 200, 128)), rtol=0, atol=0, equal_nan=True)


# ---------------------------------------------------------------------------
# Grouped product
# ---------------------------------------------------------------------------
def segments(counts):
    pad = [-(-c // 128) * 128 for c in counts]
    start = [0]
    for c in pad:
        start.append(start[-1] + c)
    dev = "cuda"
    return (torch.tensor(start, dtype=torch.int32, device=dev), torch.tensor(counts, dtype=torch.int32, device=dev), start)


def check_product(counts, N, K, out_dtype, relu, mode, seed=0, extra=0, bias=True):
    G = len(counts)
    seg, cnt, start = segments(counts)
    R = start[-1] + extra
    a = ops.quantize_fp8(acts(R, K, seed + 1))
    w = ops.quantize_fp8_weight(weight(G, N, K, seed + 2))
    b = torch.randn(G, N, generator=gen(seed + 3), device="cuda") * 0.3 if bias else None
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = 7.0 if out_dtype != torch.float8_e4m3fn else None
    out = torch.full((R, N), keep, dtype=out_dtype, device="cuda") if keep else None
    y = ops.grouped_gemm_fp8(a, w, b, relu=relu, seg_start=seg, counts=cnt, out_dtype=out_dtype, mode=mode, out=out, err=err)
    assert _lib.read_device_error(err) == 0
    av, wv = fo.read(a), fo.read(w)
    got = (fo.read(y) if out_dtype == torch.float8_e4m3fn else y).double()
    parts = fo.product(av, wv, b, relu, [(start[g], start[g] + counts[g]) for g in range(G)])
    for g, (ref, mag) in enumerate(parts):
        r0, r1 = start[g], start[g] + counts[g]
        e = fo.sum_error(mag, K)
        if out_dtype == torch.float8_e4m3fn:
            tol = fo.ambiguous(ref, e) if counts[g] else e
            ref = fo.values(*fo.quantize(ref)) if counts[g] else ref
        else:
            tol = e + HALF[out_dtype] * (ref.abs() + e)
        diff = (got[r0:r1] - ref).abs()
        assert bool((diff <= tol).all()), (g, float((diff - tol).max()), float(diff.max()))
        assert int((got[r1:start[g + 1]] != 0).sum()) == 0          # rows behind the count
    if keep and extra:
        assert bool((y[start[-1]:] == keep).all())                  # rows of no group are left alone


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
@pytest.mark.parametrize("rows,N,K", [(1, 16, 16), (1, 128, 128), (5, 144, 528), (33, 272, 1280), (128, 256, 512),
                                      (300, 400, 640), (257, 3200, 1280)])
def test_product_dense(rows, N, K, mode):
    a = ops.quantize_fp8(acts(rows, K, 5))
    w = ops.quantize_fp8_weight(weight(1, N, K, 6))
    bias = torch.randn(1, N, generator=gen(7), device="cuda")
    y = ops.grouped_gemm_fp8(a, w, bias, mode=mode)
    (ref, mag), = fo.product(fo.read(a), fo.read(w), bias, False, [(0, rows)])
    e = fo.sum_error(mag, K)
    assert bool(((y.double() - ref).abs() <= e + HALF[torch.bfloat16] * (ref.abs() + e)).all())


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("counts,N,K", [([0, 1, 0, 129, 31, 0], 144, 272), ([128, 256, 127, 300], 640, 1280),
                                        ([40] * 20, 272, 528), ([513, 2], 384, 144)])
def test_product_grouped(counts, N, K, out_dtype, mode):
    check_product(counts, N, K, out_dtype, True, mode, seed=len(counts), extra=256)


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
def test_product_no_rows_at_all(mode):
    check_product([0, 0, 0], 128, 128, torch.bfloat16, False, mode, extra=128)


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
def test_product_without_bias_and_many_groups(mode):
    g = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 9, (512,), generator=g).tolist()
    check_product(counts, 128, 256, torch.float16, False, mode, bias=False)


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
def test_product_long(mode):
    """Several waves of units on every SM, and many k-blocks."""
    check_product([3000, 1, 2047, 900], 1280, 3200, torch.bfloat16, False, mode)


def test_product_auto_choices_agree():
    """The two kernels multiply and add the same terms; their results differ by the order of the sums at most."""
    for counts in ([20] * 8, [100] * 8, [700] * 3):
        check_product(counts, 384, 640, torch.bfloat16, True, _lib.AGM_FP8_AUTO)


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
def test_product_keeps_nan(mode):
    """A NaN activation reaches its own row only, through the ReLU."""
    x = acts(200, 256, 9)
    x[7, 5] = float("nan")
    a, w = ops.quantize_fp8(x), ops.quantize_fp8_weight(weight(1, 128, 256, 10))
    y = ops.grouped_gemm_fp8(a, w, relu=True, mode=mode)
    assert bool(torch.isnan(y[7]).all()) and int(torch.isnan(y).any(1).sum()) == 1


@pytest.mark.parametrize("mode", [WEIGHTS, ROWS])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_product_rows_that_end_inside_a_tile(out_dtype, mode):
    """The last segment's 128 rows need not all exist: nothing is written behind the last row."""
    counts, R, N, K = [130, 3, 70], 640 - 57, 144, 256
    seg, cnt, start = segments(counts)
    a, w = ops.quantize_fp8(acts(R, K, 1)), ops.quantize_fp8_weight(weight(3, N, K, 2))
    assert start[2] + counts[2] < R < start[3] + 128
    seg[2], cnt[2] = 512, R - 512                              # the last segment holds the last row
    for last in (R - 512, 3):
        cnt[2] = last
        big = torch.full((R + 200, N), 5, dtype=torch.uint8, device="cuda")
        if out_dtype == torch.bfloat16:
            big = big.to(out_dtype)
        out = big.view(out_dtype)[:R]
        y = ops.grouped_gemm_fp8(a, w, seg_start=seg, counts=cnt, out_dtype=out_dtype, mode=mode, out=out)
        got = (fo.read(y) if out_dtype == torch.float8_e4m3fn else y).double()
        assert bool((big[R:] == 5).all())
        assert bool((got[512 + last:] == 0).all()) and bool((got[512:512 + last] != 0).any(1).all())


def test_product_bad_segments_are_left_out():
    """Segments that leave the rows, or do not start at a tile, are refused on the device: the others are computed."""
    a, w = ops.quantize_fp8(acts(384, 128, 1)), ops.quantize_fp8_weight(weight(3, 128, 128, 2))
    cnt = torch.tensor([10, 10, 10], dtype=torch.int32, device="cuda")
    for mode in (WEIGHTS, ROWS):
        for bad in (64, 384, -128, 2 ** 30):
            seg = torch.tensor([0, bad, 256, 384], dtype=torch.int32, device="cuda")
            err = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = torch.full((384, 128), 3.0, dtype=torch.bfloat16, device="cuda")
            ops.grouped_gemm_fp8(a, w, seg_start=seg, counts=cnt, mode=mode, out=out, err=err)
            assert _lib.read_device_error(err) == 2
            assert bool((out[128:256] == 3).all()) and bool((out[:10] != 3).any()) and bool((out[256:266] != 3).any())


def test_offsets_past_32_bits():
    """More than 2^31 elements: the end comes out as it does on its own."""
    R, W, N = 1_700_001, 1296, 1312
    x = torch.empty(R, W, dtype=torch.bfloat16, device="cuda").normal_(generator=gen(1))
    s = R // 128 * 128 - 1280
    q, p = ops.quantize_fp8(x), ops.quantize_fp8(x[s:].contiguous())
    assert torch.equal(q.q[s:].view(torch.uint8), p.q.view(torch.uint8)) and torch.equal(q.scales[s // 128:], p.scales)
    assert torch.equal(ops.dequantize_fp8(q)[s:], ops.dequantize_fp8(p))
    w = ops.quantize_fp8_weight(weight(1, N, W, 2))
    for mode in (ROWS, WEIGHTS):
        assert torch.equal(ops.grouped_gemm_fp8(q, w, mode=mode)[s:], ops.grouped_gemm_fp8(p, w, mode=mode))
        y, z = (ops.grouped_gemm_fp8(t, w, mode=mode, out_dtype=torch.float8_e4m3fn) for t in (q, p))
        assert torch.equal(y.q[s:].view(torch.uint8), z.q.view(torch.uint8)) and torch.equal(y.scales[s // 128:], z.scales)
        del y, z
    del q, p
    n, E, d, H = 1_100_000, 16, 1024, 256
    x = x.view(-1)[:n * d].view(n, d)
    idx, wgt = ops.route_experts(torch.randn(n, E, generator=gen(3), device="cuda"), 2)
    wts = make_experts(E, d, H, 4)
    out = ops.moe_experts_fp8(x, idx, wgt, *wts, check_errors=True)
    tail = (t[-4000:].contiguous() for t in (x, idx, wgt))
    assert torch.equal(out[-4000:], ops.moe_experts_fp8(*tail, *wts))


# ---------------------------------------------------------------------------
# The experts' forward
# ---------------------------------------------------------------------------
def make_experts(E, d, H, seed):
    w1 = ops.quantize_fp8_weight(weight(E, H, d, seed))
    w2 = ops.quantize_fp8_weight(weight(E, d, H, seed + 1))
    b1 = torch.randn(E, H, generator=gen(seed + 2), device="cuda") * 0.2
    b2 = torch.randn(E, d, generator=gen(seed + 3), device="cuda") * 0.2
    return w1, b1, w2, b2


def check_experts(n, E, k, d, H, dtype, seed=0, drop=0.0, residual=False, idx=None):
    x = acts(n, d, seed + 10, dtype)
    wts = make_experts(E, d, H, seed + 20)
    if idx is None:
        idx, wgt = ops.route_experts(torch.randn(n, E, generator=gen(seed + 30), device="cuda"), k)
    else:
        wgt = torch.rand(idx.shape, generator=gen(seed + 31), device="cuda") - 0.3
    if drop:
        idx = torch.where(torch.rand(n, k, generator=gen(seed + 32), device="cuda") < drop, torch.full_like(idx, -1), idx)
    res = acts(n, d, seed + 33, dtype) if residual else None
    out = ops.moe_experts_fp8(x, idx, wgt, *wts, residual=res, check_errors=True)
    ref, tol = fo.experts(x.double(), idx, wgt, fo.read(wts[0]), wts[1], fo.read(wts[2]), wts[3], HALF[dtype], res)
    diff = (out.double() - ref).abs()
    assert bool((diff <= tol).all()), float((diff / tol.clamp_min(1e-30)).max())
    return x, idx, wgt, wts, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,E,k,d,H", [(1, 4, 1, 16, 16), (1, 64, 8, 256, 144), (7, 3, 3, 144, 272), (64, 14, 2, 1280, 3200),
                                       (200, 100, 5, 272, 400), (1500, 14, 2, 528, 640), (2999, 20, 6, 256, 384)])
def test_experts(n, E, k, d, H, dtype):
    check_experts(n, E, k, d, H, dtype, seed=n)


def test_experts_many():
    check_experts(700, 512, 8, 128, 144, torch.bfloat16, seed=1)
    check_experts(40, 512, 32, 128, 144, torch.bfloat16, seed=2)


@pytest.mark.parametrize("n", [50, 3000])
def test_experts_dropped_slots_and_residual(n):
    x, idx, wgt, wts, out = check_experts(n, 9, 4, 256, 384, torch.bfloat16, seed=n, drop=0.4, residual=True)
    # a token without any expert keeps its residual, or gets zeros
    idx = torch.full_like(idx, -1)
    assert int(ops.moe_experts_fp8(x, idx, wgt, *wts, check_errors=True).count_nonzero()) == 0
    assert torch.equal(ops.moe_experts_fp8(x, idx, wgt, *wts, residual=x, check_errors=True), x)


@pytest.mark.parametrize("n", [30, 1000])
def test_experts_repeated_and_foreign_indices(n):
    """The same expert twice in a row counts twice; indices outside [0, E) go nowhere."""
    idx = torch.randint(-3, 8, (n, 4), generator=gen(4), device="cuda", dtype=torch.int32)
    idx[:, 1] = idx[:, 0]
    idx[::3, 2] = 6
    check_experts(n, 6, 4, 256, 128, torch.float16, seed=n, idx=idx)


@pytest.mark.parametrize("n", [100, 5000])
def test_experts_all_on_one(n):
    idx = torch.full((n, 1), 3, dtype=torch.int32, device="cuda")
    check_experts(n, 8, 1, 256, 272, torch.bfloat16, seed=n, idx=idx)


def test_experts_no_tokens():
    wts = make_experts(4, 64, 128, 1)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    out = ops.moe_experts_fp8(x, torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                              torch.empty(0, 2, device="cuda"), *wts, check_errors=True)
    assert out.shape == (0, 64)


def test_experts_same_as_the_stages():
    """One call equals quantise, product, product and weighted sum by hand, where a token has one expert."""
    n, d, H = 300, 256, 384
    wts = make_experts(1, d, H, 5)
    x = acts(n, d, 6, torch.bfloat16)
    idx = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    out = ops.moe_experts_fp8(x, idx, torch.ones(n, 1, device="cuda"), *wts, check_errors=True)
    h = ops.grouped_gemm_fp8(ops.quantize_fp8(x), wts[0], wts[1], relu=True, out_dtype=torch.float8_e4m3fn, mode=ROWS)
    assert torch.equal(out, ops.grouped_gemm_fp8(h, wts[2], wts[3], mode=ROWS))


def test_experts_repeatable_on_streams_and_in_graphs():
    """Bit-identical when run twice, on two streams at once, and captured twice and replayed at once."""
    n, E, k, d, H = 777, 12, 3, 512, 640
    wts = make_experts(E, d, H, 1)
    xs = [acts(n, d, 2 + i, torch.bfloat16) for i in range(2)]
    idx, wgt = ops.route_experts(torch.randn(n, E, generator=gen(9), device="cuda"), k)
    ref = [ops.moe_experts_fp8(x, idx, wgt, *wts, check_errors=True) for x in xs]
    assert torch.equal(ref[0], ops.moe_experts_fp8(xs[0], idx, wgt, *wts))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    outs = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            outs.append(ops.moe_experts_fp8(x, idx, wgt, *wts))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    graphs, gouts = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gouts.append(ops.moe_experts_fp8(x, idx, wgt, *wts))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(gouts, ref))


@pytest.mark.parametrize("n", [1, 40, 200])
def test_small_batches_at_once(n):
    """Both products in one launch, several such launches at a time on streams and in graphs."""
    E, k, d, H = 14, 2, 512, 640
    wts = make_experts(E, d, H, 1)
    xs = [acts(n, d, 2 + i, torch.bfloat16) for i in range(4)]
    route = [ops.route_experts(torch.randn(n, E, generator=gen(9 + i), device="cuda"), k) for i in range(4)]
    ref = [ops.moe_experts_fp8(x, *r, *wts, check_errors=True) for x, r in zip(xs, route)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        outs = []
        for s, x, r in zip(streams, xs, route):
            with torch.cuda.stream(s):
                outs.append(ops.moe_experts_fp8(x, *r, *wts))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    graphs, gouts = [], []
    for x, r in zip(xs, route):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gouts.append(ops.moe_experts_fp8(x, *r, *wts))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(gouts, ref))


@pytest.mark.parametrize("n", [1, 64, 900])
def test_one_workspace_for_calls_in_a_row(n):
    """Launches overlap at their ends: another routing in the same workspace must not show through."""
    E, k, d, H = 14, 2, 256, 384
    wts = make_experts(E, d, H, 1)
    x = acts(n, d, 2, torch.bfloat16)
    route = [ops.route_experts(torch.randn(n, E, generator=gen(9 + i), device="cuda"), k) for i in range(3)]
    ref = [ops.moe_experts_fp8(x, *r, *wts, check_errors=True) for r in route]
    nbytes = _lib.load().agm_moe_experts_fp8_workspace_bytes(n, d, E, k, H)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    outs = [ops.moe_experts_fp8(x, *route[i % 3], *wts, workspace=ws) for i in range(60)]
    assert all(torch.equal(o, ref[i % 3]) for i, o in enumerate(outs))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [ops.moe_experts_fp8(x, *route[i % 3], *wts, workspace=ws) for i in range(12)]
    for _ in range(5):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i % 3]) for i, o in enumerate(outs))


@pytest.mark.parametrize("top_k,shared,residual", [(1, 0, False), (2, 0, True), (2, 2, True), (3, 1, False)])
def test_module_with_8_bit_experts(top_k, shared, residual):
    """MoEFFN with expert_precision "fp8" against the same routing through the definition; a changed parameter is seen."""
    torch.manual_seed(3)
    d, E, n, dtype = 256, 6, 150, torch.bfloat16
    m = agillm41_b200.MoEFFN(d, mlp_mult=2, experts=E, top_k=top_k, shared_experts=shared, shared_mlp_mult=1)
    for blk in (m.shared or []):
        torch.nn.init.normal_(blk[2].weight, std=0.05)
        torch.nn.init.normal_(blk[2].bias, std=0.1)
    m = m.to(device="cuda", dtype=dtype).eval()
    m.check_device_errors = True
    x = acts(n, d, 4, dtype).view(3, 50, d)
    res = acts(n, d, 5, dtype).view(3, 50, d) if residual else None
    with torch.no_grad():
        plain = m.forward_residual(x, res) if residual else m(x)
        m.expert_precision = "fp8"
        for step in range(2):
            got = m.forward_residual(x, res) if residual else m(x)
            idx, gates, _, _ = ops.router_topk(x.view(n, d), m.router.weight.contiguous(), top_k)

            def q(mods, i):
                return fo.read(ops.quantize_fp8_weight(torch.stack([ex[i].weight for ex in mods])))

            def b(mods, i):
                return torch.stack([ex[i].bias for ex in mods]).float()

            add = None if res is None else res.view(n, d).double()
            slack = 0.0
            for blk in (m.shared or []):
                y, t = fo.experts(x.view(n, d).double(), torch.zeros(n, 1, dtype=torch.int32, device="cuda"),
                                  torch.ones(n, 1, device="cuda"), q([blk], 0), b([blk], 0), q([blk], 2), b([blk], 2), HALF[dtype])
                # the sum with what came before is rounded to the activation type
                add = y if add is None else add + y
                slack = slack + t + HALF[dtype] * add.abs()
            ref, tol = fo.experts(x.view(n, d).double(), idx, gates.float(), q(m.experts, 0), b(m.experts, 0), q(m.experts, 2),
                                  b(m.experts, 2), HALF[dtype], add)
            assert bool(((got.view(n, d).double() - ref).abs() <= tol + slack * (1 + HALF[dtype])).all())
            m.experts[0][0].weight.mul_(1.5)
            m.experts[1][2].bias.add_(0.5)
        m.expert_precision = "model"
        assert plain.shape == got.shape and not torch.equal(plain, got)
    m.expert_precision = "fp8"
    with pytest.raises(agillm41_b200.MoEKernelError):
        m(x)                                                   # gradients wanted
    with torch.no_grad(), pytest.raises(agillm41_b200.MoEKernelError):
        m.expert_precision = "int3"
        m(x)


def test_module_8_bit_copies_follow_the_parameters():
    """Captured, replayed after a change, first run in inference mode, with replaced parameters."""
    torch.manual_seed(5)
    d, E, n, dtype = 256, 4, 40, torch.bfloat16
    x = acts(n, d, 4, dtype)

    def module():
        m = agillm41_b200.MoEFFN(d, mlp_mult=2, experts=E, top_k=2, shared_experts=1, shared_mlp_mult=1)
        m = m.to(device="cuda", dtype=dtype).eval()
        m.expert_precision = "fp8"
        return m

    def fresh(m):
        c = module()
        c.load_state_dict(m.state_dict())
        return c(x)

    m = module()
    with torch.no_grad():
        with pytest.raises(agillm41_b200.MoEKernelError):      # nothing to capture yet
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                m(x)
        first = m(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m(x)
        g.replay()
        assert torch.equal(out, first)
        m.experts[1][0].weight.mul_(1.5)
        m.shared[0][2].bias.add_(0.5)
        got = m(x)
        assert not torch.equal(got, first) and torch.equal(got, fresh(m))
        g.replay()                                             # reads the same memory
        assert torch.equal(out, got)
        for _ in range(3):                                     # new parameters, perhaps at an old one's address
            m.experts[2][2].weight = torch.nn.Parameter(torch.randn(d, 2 * d, device="cuda").to(dtype) * 0.05)
            assert torch.equal(m(x), fresh(m))
    m = module()
    with torch.inference_mode():
        first = m(x).clone()
    with torch.no_grad():
        assert torch.equal(m(x), first)
        m.experts[0][0].bias.add_(0.5)
        assert torch.equal(m(x), fresh(m)) and not torch.equal(m(x), first)
        m.router.weight.mul_(0.5)
    with torch.inference_mode():
        assert torch.equal(m(x), fresh(m))


def test_module_8_bit_copies_on_two_streams():
    """First used on a busy stream, then at once on another; no tokens at all; copied and pickled."""
    torch.manual_seed(6)
    d, E, n, dtype = 1024, 8, 64, torch.bfloat16
    m = agillm41_b200.MoEFFN(d, mlp_mult=2, experts=E, top_k=2).to(device="cuda", dtype=dtype).eval()
    m.expert_precision = "fp8"
    x = acts(n, d, 4, dtype)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    with torch.no_grad():
        m._packed_weights(x.device, dtype)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            for _ in range(20):
                busy = busy @ busy * 1e-4
            first = m(x)
        with torch.cuda.stream(b):
            second = m(x)
        torch.cuda.synchronize()
        assert torch.equal(first, m(x)) and torch.equal(second, first)
        assert m(x[:0]).shape == (0, d)
        twin = copy.deepcopy(m)
        twin.experts[0][0].weight.mul_(2)
        assert not torch.equal(twin(x), first) and torch.equal(m(x), first)
        blob = io.BytesIO()
        torch.save(m, blob)
        blob.seek(0)
        assert torch.equal(torch.load(blob, weights_only=False)(x), first)


def test_torch_operators_match():
    n, E, k, d, H = 70, 9, 3, 144, 272
    x = acts(n, d, 1, torch.float16)
    w1, b1, w2, b2 = make_experts(E, d, H, 2)
    o = torch.ops.agillm_moe
    idx, wgt = o.route_experts(torch.randn(n, E, generator=gen(3), device="cuda"), k, "softmax", None, 1, 1, True, 1.0)
    y = o.moe_experts_fp8(x, idx, wgt, *w1, b1, *w2, b2, x)
    assert torch.equal(y, ops.moe_experts_fp8(x, idx, wgt, w1, b1, w2, b2, residual=x))
    q = o.quantize_fp8(x)
    assert torch.equal(o.dequantize_fp8(*q, torch.float32), ops.dequantize_fp8(ops.quantize_fp8(x), torch.float32))
    one = ops.FP8Tensor(w1.q[:1].contiguous(), w1.scales[:1].contiguous())
    assert torch.equal(o.grouped_gemm_fp8(*q, *one, b1[:1], True, None, None, torch.float16),
                       ops.grouped_gemm_fp8(ops.FP8Tensor(*q), one, b1[:1], relu=True, out_dtype=torch.float16))


def test_quantize_weight_into():
    w = weight(3, 80, 272, 1).bfloat16()
    out = ops.quantize_fp8_weight(weight(3, 80, 272, 2))
    again = ops.quantize_fp8_weight(w, out=out)
    ref = ops.quantize_fp8_weight(w)
    assert again.q.data_ptr() == out.q.data_ptr()
    assert torch.equal(again.q.view(torch.uint8), ref.q.view(torch.uint8)) and torch.equal(again.scales, ref.scales)
    with pytest.raises(agillm41_b200.MoEKernelError):
        ops.quantize_fp8_weight(w[:2], out=out)


def test_refusals_on_the_gpu():
    E = agillm41_b200.MoEKernelError
    x = acts(8, 64, 1, torch.bfloat16)
    a, w = ops.quantize_fp8(x), ops.quantize_fp8_weight(weight(2, 32, 64, 2))
    with pytest.raises(E):
        ops.quantize_fp8(acts(8, 24, 1))                       # width no multiple of 16
    with pytest.raises(E):
        ops.quantize_fp8(x.t())                                # not contiguous
    with pytest.raises(E):
        ops.quantize_fp8(x[0])                                 # one dimension
    with pytest.raises(E):
        ops.quantize_fp8_weight(x)
    with pytest.raises(E):
        ops.quantize_fp8(x.to(torch.int32))
    with pytest.raises(E):
        ops.grouped_gemm_fp8(a, w)                             # two groups without segments
    seg, cnt, _ = segments([4, 4])
    with pytest.raises(E):
        ops.grouped_gemm_fp8(a, w, seg_start=seg)
    with pytest.raises(E):
        ops.grouped_gemm_fp8(a, w, seg_start=seg.long(), counts=cnt)
    with pytest.raises(E):
        ops.grouped_gemm_fp8(a, w, seg_start=seg, counts=cnt, out_dtype=torch.float32)
    with pytest.raises(E):
        ops.grouped_gemm_fp8(a, w, torch.zeros(2, 32, device="cuda", dtype=torch.bfloat16), seg_start=seg, counts=cnt)
    with pytest.raises(E):
        ops.grouped_gemm_fp8(ops.FP8Tensor(a.q, a.scales[:, :, :256].contiguous()), w, seg_start=seg, counts=cnt)
    with pytest.raises(E):
        ops.grouped_gemm_fp8(x, w, seg_start=seg, counts=cnt)
    w1, b1, w2, b2 = make_experts(3, 64, 128, 1)
    idx = torch.zeros(8, 2, dtype=torch.int32, device="cuda")
    wgt = torch.zeros(8, 2, device="cuda")
    with pytest.raises(E):
        ops.moe_experts_fp8(x.float(), idx, wgt, w1, b1, w2, b2)
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx.long(), wgt, w1, b1, w2, b2)
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx, wgt[:4], w1, b1, w2, b2)
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx, wgt, w2, b1, w1, b2)
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx, wgt, w1, b1, w2, b2.bfloat16())
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx, wgt, w1, b1, w2, b2, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(E):
        ops.moe_experts_fp8(x, idx, wgt, w1, b1.cpu(), w2, b2)
