"""Definition of the block-scaled e4m3 format and of the products over it, in 64 bits.

Test infrastructure only. Values are float64 tensors on any device; nothing
here uses torch's 8-bit types except to read and write their bytes.
"""
import torch

BLOCK = 128


def round_e4m3(v):
    """Nearest e4m3 value of |v| <= 448, ties to even: 3 mantissa bits down to 2^-6, steps of 2^-9 below."""
    _, e = torch.frexp(v)                       # |v| = m * 2^e, m in [0.5, 1)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9).to(torch.int32))
    return torch.round(v / step) * step         # torch.round: half to even


def e4m3_step(v):
    _, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9).to(torch.int32))


def exponent(amax):
    """Least p >= -127 with amax <= 448 * 2^p."""
    p = torch.full(amax.shape, -127.0, dtype=torch.float64, device=amax.device)
    pos = amax > 0
    m, e = torch.frexp(amax)
    p = torch.where(pos, (e - 9).double() + (m > 0.875), p)
    return p.clamp_min(-127)


def _blocks(x, br):
    """[..., rows, width] -> zero-padded [..., R, br, C, 128]."""
    rows, width = x.shape[-2:]
    R, C = -(-rows // br), -(-width // BLOCK)
    full = x.new_zeros(*x.shape[:-2], R * br, C * BLOCK)
    full[..., :rows, :width] = x
    return full.view(*x.shape[:-2], R, br, C, BLOCK)


def quantize(x, block_rows=1):
    """x [..., rows, width] float64 -> (values of q, exponents [..., ceil(rows / block_rows), blocks])."""
    rows, width = x.shape[-2:]
    b = _blocks(x, block_rows)
    finite = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b))
    p = exponent(finite.amax(dim=(-3, -1)))
    s = torch.exp2(p)[..., :, None, :, None]
    q = torch.where(torch.isfinite(b), round_e4m3(b / s), torch.full_like(b, float("nan")))
    lead = x.shape[:-2]
    return q.reshape(*lead, b.shape[-4] * block_rows, -1)[..., :rows, :width], p


def row_exponents(p, rows, block_rows):
    return p.repeat_interleave(block_rows, dim=-2)[..., :rows, :]


def values(q, p_rows):
    """q [..., rows, width] and exponents per row [..., rows, blocks] -> what they stand for, float64."""
    return q.double() * torch.exp2(p_rows.double()).repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def tiles_of(p_rows):
    """Exponents per row [rows, blocks] -> scale tiles uint8 [ceil(rows/128), ceil(blocks/4), 512], one byte at a time."""
    rows, blocks = p_rows.shape
    out = torch.zeros(-(-rows // 128), -(-blocks // 4), 512, dtype=torch.uint8)
    r = torch.arange(rows)[:, None].expand(rows, blocks)
    b = torch.arange(blocks)[None, :].expand(rows, blocks)
    out[r // 128, b // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4] = (p_rows.cpu() + 127).to(torch.uint8)
    return out


def exponents_of(tiles, rows, blocks):
    """Scale tiles [T, K4, 512] -> exponents per row [rows, blocks]."""
    r = torch.arange(rows, device=tiles.device)[:, None].expand(rows, blocks)
    b = torch.arange(blocks, device=tiles.device)[None, :].expand(rows, blocks)
    return tiles[r // 128, b // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4].double() - 127


def read(t):
    """FP8Tensor -> float64 values."""
    rows, width = t.q.shape[-2:]
    blocks = -(-width // BLOCK)
    if t.q.dim() == 2:
        return values(t.q.float(), exponents_of(t.scales, rows, blocks))
    return torch.stack([values(t.q[g].float(), exponents_of(t.scales[g], rows, blocks)) for g in range(t.q.shape[0])])


def product(a, w, bias, relu, row_slices):
    """[(act(a w_g^T + b_g), sum of |terms|)] per group; a [R, K], w [G, N, K] float64, row_slices [(r0, r1)]."""
    out = []
    for g, (r0, r1) in enumerate(row_slices):
        y = a[r0:r1] @ w[g].t()
        mag = a[r0:r1].abs() @ w[g].abs().t()
        if bias is not None:
            y, mag = y + bias[g].double(), mag + bias[g].double().abs()
        out.append((torch.relu(y) if relu else y, mag))
    return out


def sum_error(mag, K):
    """Bound on the error of an fp32 sum of K exact products and a bias: every
    tensor-core step (32 products and the running sum) and the bias add is off
    by at most 2^-22 of the sum of the magnitudes."""
    return mag * (K / 32 + 1) * 2.0 ** -22


def ambiguous(v, err):
    """For values v [rows, width] known to within err: how far the requantised value may be from the one
    quantize(v) gives: one step where v is that near to a rounding border, a step everywhere in a block whose
    maximum is that near to a change of the scale."""
    rows, width = v.shape
    q, p = quantize(v)
    s = torch.exp2(p).repeat_interleave(BLOCK, -1)[:, :width]
    u, e = v / s, err / s
    lo, hi = round_e4m3((u - e).clamp(-448, 448)), round_e4m3((u + e).clamp(-448, 448))
    slack = torch.where(lo != hi, e4m3_step(u) * s, torch.zeros_like(u))
    amax = _blocks(v.abs(), 1).amax(dim=(-3, -1))
    emax = _blocks(err, 1).amax(dim=(-3, -1))
    edge = exponent((amax - emax).clamp_min(0)) != exponent(amax + emax)
    wide = edge.repeat_interleave(BLOCK, -1)[:, :width]
    return torch.where(wide, 2 * e4m3_step(u) * s, slack) + err


def experts(x, idx, weights, w1, b1, w2, b2, half_step, residual=None):
    """The experts' forward -> (out, tolerance): float64 x [N, d], w1 [E, H, d], w2 [E, d, H] as values.
    half_step: half a step of the activation type, relative."""
    n, d = x.shape
    E, H = w1.shape[:2]
    q, p = quantize(x)
    xq = values(q, p)
    out = torch.zeros_like(x) if residual is None else residual.double().clone()
    tol = torch.zeros_like(x)
    mag = out.abs()
    for e in range(E):
        tok, rank = torch.nonzero(idx == e, as_tuple=True)
        if not tok.numel():
            continue
        (h, hm), = product(xq[tok], w1[e:e + 1], b1[e:e + 1], True, [(0, tok.numel())])
        slack = ambiguous(h, sum_error(hm, d))
        hq = values(*quantize(h))
        (y, ym), = product(hq, w2[e:e + 1], b2[e:e + 1], False, [(0, tok.numel())])
        ye = slack @ w2[e].abs().t() + sum_error(ym, H)
        ye = ye + half_step * (y.abs() + ye)          # y is rounded to the activation type
        g = weights[tok, rank].double()[:, None]
        out.index_add_(0, tok, g * y)
        tol.index_add_(0, tok, g.abs() * ye)
        mag.index_add_(0, tok, g.abs() * y.abs())
    k = idx.shape[1]
    tol = tol + mag * (k + 1) * 2.0 ** -24            # the fp32 weighted sum
    return out, tol + half_step * (out.abs() + tol)   # the output's own rounding
