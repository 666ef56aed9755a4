"""Workloads of the general expert router and of the 8-bit floating point expert path.

Four operators, each a public entry point of ``agillm41_b200.ops``:

* ``route``     ``route_experts`` / ``route_experts_backward``: softmax or sigmoid scores of router logits,
                a selection bias, groups of experts, top-k, renormalised and scaled weights
* ``quantize``  ``quantize_fp8`` / ``quantize_fp8_weight`` and ``dequantize_fp8``: e4m3 values with one
                power-of-two scale per block of 128 (1 x 128 for rows, 128 x 128 for weights), and back
* ``product``   ``grouped_gemm_fp8``: act(a @ w[g]^T + bias[g]) over expert segments of block-scaled rows
* ``experts``   ``moe_experts_fp8``: the routed experts of a MoE block with 8-bit weights (dispatch,
                quantisation, FC1 + ReLU + requantisation, FC2, weighted sum)

``run`` computes them in plain torch operations, or, where ``own`` is set, by the package's calls.
"""
import math

import torch

own = False

BLOCK = 128          # elements that share one scale
E4M3_MAX = 448.0     # largest e4m3 value
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One decode step of the repository's 14-expert block: 64 sequences, top-2. Latency counts.
        dict(name="route decode", op="route", n=64, e=14, k=2, score="softmax", bias=False, groups=1, keep=1,
             renorm=True, scale=1.0, dtype="fp32", train=False),
        # Prompt processing with many experts: sigmoid scores, balance bias, half of 8 groups kept, top-8.
        dict(name="route prompt grouped", op="route", n=65536, e=256, k=8, score="sigmoid", bias=True, groups=8, keep=4,
             renorm=True, scale=2.5, dtype="fp32", train=False),
        # A training step's routing, forward and gradient, weights not renormalised (every logit has a gradient).
        dict(name="route train", op="route", n=49151, e=64, k=6, score="softmax", bias=False, groups=1, keep=1,
             renorm=False, scale=1.0, dtype="bf16", train=True),
        # The activations of the benchmark batch (48 x 1536 tokens, width 1280), quantised and read back.
        dict(name="quantize rows", op="quantize", kind="rows", g=1, n=73728, width=1280, dtype="bf16"),
        # The first expert matrices of one layer, quantised when a checkpoint is loaded, and read back.
        dict(name="quantize weights", op="quantize", kind="weights", g=14, n=3200, width=1280, dtype="bf16"),
        # One token through one dense matrix: the smallest product, bound by latency.
        dict(name="product one token", op="product", g=1, rows=1, n=3200, width=1280, relu=False, dtype="bf16"),
        # A small ragged batch over many experts, some without rows, odd widths.
        dict(name="product ragged", op="product", g=61, rows=1999, n=1488, width=2000, relu=True, dtype="fp16"),
        # The second expert product of the benchmark batch: 147,456 rows over 14 experts, skewed.
        dict(name="product prompt", op="product", g=14, rows=147456, n=1280, width=3200, relu=False, dtype="bf16"),
        # The experts of one decode step (64 tokens, top-2 of 14): bound by reading the weights.
        dict(name="experts decode", op="experts", n=64, e=14, k=2, width=1280, hidden=3200, drop=0.0, dtype="bf16"),
        # A single token, top-8 of 64 narrow experts.
        dict(name="experts one token", op="experts", n=1, e=64, k=8, width=2048, hidden=1408, drop=0.0, dtype="bf16"),
        # A mid-size padded batch (a twelfth of the slots routed nowhere), odd token count.
        dict(name="experts padded", op="experts", n=2999, e=64, k=6, width=2048, hidden=1408, drop=0.08, dtype="fp16"),
        # The benchmark batch: 73,728 tokens, top-2 of 14 experts.
        dict(name="experts prompt", op="experts", n=73728, e=14, k=2, width=1280, hidden=3200, drop=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "quantize", "product", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * max(2, _log(rng, 4, 256) // groups)
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(8, e // groups * keep))
        return dict(op=op, n=_log(rng, 1, 65536), e=e, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, keep=keep, renorm=rng.random() < 0.5,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    train=rng.random() < 0.5)
    if op == "quantize":
        kind = rng.choice(["rows", "weights"])
        width = 16 * _log(rng, 4, 256)
        if kind == "rows":
            return dict(op=op, kind=kind, g=1, n=_log(rng, 1, min(65536, 90_000_000 // width)), width=width,
                        dtype=rng.choice(list(DTYPES)))
        return dict(op=op, kind=kind, g=_log(rng, 1, 16), n=16 * _log(rng, 4, 200), width=min(width, 1600),
                    dtype=rng.choice(list(DTYPES)))
    width, n = 16 * _log(rng, 8, 200), 16 * _log(rng, 8, 200)
    if op == "product":
        rows = _log(rng, 1, min(131072, int(5.0e11) // (n * width)))
        return dict(op=op, g=_log(rng, 1, 64), rows=rows, n=n, width=width, relu=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "fp16"]))
    e = _log(rng, 2, 64)
    k = rng.randint(1, min(8, e))
    tokens = _log(rng, 1, max(2, min(65536, int(4.0e11) // (n * width * k))))
    return dict(op=op, n=tokens, e=e, k=k, width=width, hidden=n, drop=rng.choice([0.0, 0.0, 0.1]),
                dtype=rng.choice(["bf16", "fp16"]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _logits(n, e, gen, dev):
    """Router logits: a spread per token and a standing preference per expert."""
    return torch.randn(n, e, generator=gen, device=dev) * 1.3 + torch.randn(e, generator=gen, device=dev) * 0.5


def _acts(n, width, gen, dev):
    """Normalised activations with a few strong channels."""
    gain = torch.exp(0.4 * torch.randn(width, generator=gen, device=dev))
    return torch.randn(n, width, generator=gen, device=dev) * gain


def _linear(g, n, width, gen, dev):
    """Weights with the spread of a freshly initialised or trained linear layer."""
    return torch.randn(g, n, width, generator=gen, device=dev) * (0.6 / math.sqrt(width))


def _exponent(amax):
    """The least p with amax <= 448 * 2^p, in [-127, 127] (amax = m * 2^e, m in [0.5, 1), 448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    p = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, p, torch.full_like(p, -127)).clamp(-127, 127)


def _padded(x, rows, width):
    return torch.nn.functional.pad(x, (0, width - x.shape[-1], 0, rows - x.shape[-2]))


def _up(v, m):
    return (v + m - 1) // m * m


def _encode_rows(x):
    """x [n, w] fp32 -> (e4m3 [n, w], exponent [n, ceil(w / 128)])."""
    n, w = x.shape
    wp = _up(w, BLOCK)
    b = _padded(x, n, wp).view(n, wp // BLOCK, BLOCK)
    p = _exponent(b.abs().amax(-1))
    q = torch.ldexp(b, -p.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q.view(n, wp)[:, :w].contiguous(), p


def _encode_weight(w):
    """w [g, n, k] fp32 -> (e4m3 [g, n, k], exponent [g, ceil(n / 128), ceil(k / 128)])."""
    g, n, k = w.shape
    np_, kp = _up(n, BLOCK), _up(k, BLOCK)
    b = _padded(w, np_, kp).view(g, np_ // BLOCK, BLOCK, kp // BLOCK, BLOCK)
    p = _exponent(b.abs().amax(dim=(2, 4)))
    q = torch.ldexp(b, -p[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(g, np_, kp)[:, :n, :k].contiguous(), p


def _per_row(p, n):
    """Exponents of 128-row blocks [.., n / 128, kb] -> of rows [.., n, kb]."""
    return p.repeat_interleave(BLOCK, dim=-2)[..., :n, :]


def _tiles(p):
    """Row exponents [.., n, kb] -> the package's scale tiles, biased by 127: uint8 [.., ceil(n / 128),
    ceil(kb / 4), 512], row r and block b of a tile at byte 16 * (r % 32) + 4 * (r / 32) + b."""
    n, kb = p.shape[-2:]
    lead = p.shape[:-2]
    t, k4 = _up(n, 128) // 128, _up(kb, 4) // 4
    b = torch.nn.functional.pad((p + 127).to(torch.uint8), (0, 4 * k4 - kb, 0, 128 * t - n))
    b = b.reshape(*lead, t, 4, 32, k4, 4)                      # tile, r / 32, r % 32, b / 4, b % 4
    d = len(lead)
    return b.permute(*range(d), d, d + 3, d + 2, d + 1, d + 4).reshape(*lead, t, k4, 512).contiguous()


def _segments(counts):
    """Row counts [g] -> starts [g + 1] of segments padded to 128 rows."""
    pad = (counts + 127) // 128 * 128
    return torch.cat([pad.new_zeros(1), pad.cumsum(0)])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    s = {"case": case}
    op = case["op"]
    if op == "route":
        s["logits"] = _logits(case["n"], case["e"], gen, dev).to(DTYPES[case["dtype"]])
        s["bias"] = torch.randn(case["e"], generator=gen, device=dev) * 0.1 if case["bias"] else None
        s["grad"] = torch.randn(case["n"], case["k"], generator=gen, device=dev) if case["train"] else None
    elif op == "quantize":
        if case["kind"] == "rows":
            x = _acts(case["n"], case["width"], gen, dev)
        else:
            x = _linear(case["g"], case["n"], case["width"], gen, dev)
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif op == "product":
        g, n, width = case["g"], case["n"], case["width"]
        if g == 1:
            s["counts"] = s["seg_start"] = None
            rows = case["rows"]
        else:
            # The split over the groups belongs to the case, so that the shapes of its outputs do.
            split = torch.Generator(device=dev)
            split.manual_seed(1000 * g + case["rows"])
            pref = torch.softmax(0.5 * torch.randn(g, generator=split, device=dev), 0)
            pick = torch.multinomial(pref, case["rows"], replacement=True, generator=split)
            counts = torch.bincount(pick, minlength=g)
            start = _segments(counts)
            rows = int(start[-1])
            s["counts"], s["seg_start"] = counts.to(torch.int32), start.to(torch.int32)
        aq, ap = _encode_rows(_acts(rows, width, gen, dev))
        wq, wp = _encode_weight(_linear(g, n, width, gen, dev))
        s["a"], s["w"] = (aq, _tiles(ap)), (wq, _tiles(_per_row(wp, n)))
        s["bias"] = torch.randn(g, n, generator=gen, device=dev) * 0.1
        s["ap"], s["wp"] = ap, wp
    else:
        n, e, k, width, hidden = (case[x] for x in ("n", "e", "k", "width", "hidden"))
        s["x"] = _acts(n, width, gen, dev).to(DTYPES[case["dtype"]])
        top = torch.topk(_logits(n, e, gen, dev), k, dim=1)
        s["idx"] = top.indices.to(torch.int32)
        if case["drop"]:
            lost = torch.rand(n, k, generator=gen, device=dev) < case["drop"]
            s["idx"] = torch.where(lost, torch.full_like(s["idx"], -1), s["idx"])
        s["weights"] = torch.softmax(top.values, dim=1)
        for name, a, b in (("1", hidden, width), ("2", width, hidden)):
            q, p = _encode_weight(_linear(e, a, b, gen, dev))
            s["w" + name], s["p" + name] = (q, _tiles(_per_row(p, a))), p
            s["b" + name] = torch.randn(e, a, generator=gen, device=dev) * 0.1
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _scores(case, logits):
    if case["score"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    z = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    return z / z.sum(dim=1, keepdim=True)


def _choose(case, logits, bias):
    """The top-k experts: selection in 64 bits, ties to the lowest index."""
    l64 = logits.double()
    s64 = _scores(case, l64)
    key = l64 if bias is None else s64 + bias.double()
    if case["keep"] < case["groups"]:
        n, groups = logits.shape[0], case["groups"]
        score = s64 if bias is None else key
        two = torch.sort(score.view(n, groups, -1), dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = torch.sort(two, dim=1, descending=True, stable=True).indices[:, :case["keep"]]
        off = torch.ones_like(two, dtype=torch.bool).scatter(1, kept, False)
        off = off.repeat_interleave(logits.shape[1] // groups, dim=1)
        key = torch.where(off, torch.full_like(key, -math.inf), key)
    return torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["k"]]


def _route(s):
    case, x = s["case"], s["logits"].float()
    idx = _choose(case, x, s["bias"])
    p = _scores(case, x)
    v = p.gather(1, idx)
    total = v.sum(dim=1, keepdim=True)
    w = (v / total if case["renorm"] else v) * case["scale"]
    if s["grad"] is None:
        return idx.to(torch.int32), w
    g = s["grad"] * case["scale"]
    if case["renorm"]:
        g = (g - (g * v).sum(dim=1, keepdim=True) / total) / total
    if case["score"] == "sigmoid":
        d = torch.zeros_like(x).scatter(1, idx, g * v * (1 - v))
    else:
        inner = 0.0 if case["renorm"] else (g * v).sum(dim=1, keepdim=True)
        d = torch.zeros_like(x).scatter(1, idx, g)
        d = p * (d - inner)
    return idx.to(torch.int32), w, d.to(s["logits"].dtype)


def _decode_rows(q, p, width):
    return torch.ldexp(q.float(), p.repeat_interleave(BLOCK, dim=-1)[..., :width])


def _decode_weight(q, p):
    return _decode_rows(q, _per_row(p, q.shape[1]), q.shape[2])


def _quantize(s):
    x = s["x"].float()
    if s["case"]["kind"] == "rows":
        return _decode_rows(*_encode_rows(x), x.shape[1]).to(s["x"].dtype)
    return _decode_weight(*_encode_weight(x)).to(s["x"].dtype)


def _slots(group, g):
    """Group of each item (g: none) -> (its place within its group, places of the largest group)."""
    order = torch.sort(group, stable=True).indices
    count = torch.bincount(group, minlength=g + 1)
    first = count.cumsum(0) - count
    place = torch.empty_like(group)
    place[order] = torch.arange(group.numel(), device=group.device) - first[group[order]]
    return place, max(1, int(count[:g].max()))


def _product(s):
    case = s["case"]
    a = _decode_rows(s["a"][0], s["ap"], case["width"])
    w = _decode_weight(s["w"][0], s["wp"])
    if s["counts"] is None:
        y = a @ w[0].t() + s["bias"][0]
        return (y.clamp_min(0) if case["relu"] else y).to(DTYPES[case["dtype"]])
    counts, start = s["counts"].long(), s["seg_start"].long()
    g, rows = case["g"], a.shape[0]
    r = torch.arange(rows, device=a.device)
    group = torch.searchsorted(start[1:].contiguous(), r, right=True).clamp_max(g - 1)
    live = r - start[group] < counts[group]
    place, most = _slots(torch.where(live, group, torch.full_like(group, g)), g)
    batch = a.new_zeros(g, most, case["width"])
    batch[group[live], place[live]] = a[live]
    y = torch.bmm(batch, w.transpose(1, 2)) + s["bias"][:, None, :]
    y = y.clamp_min(0) if case["relu"] else y
    out = torch.zeros(rows, case["n"], device=a.device)
    out[live] = y[group[live], place[live]]
    return out.to(DTYPES[case["dtype"]])


def _experts(s):
    case = s["case"]
    n, e, k, width = case["n"], case["e"], case["k"], case["width"]
    x = _decode_rows(*_encode_rows(s["x"].float()), width)
    group = s["idx"].long().reshape(-1)
    live = group >= 0
    place, most = _slots(torch.where(live, group, torch.full_like(group, e)), e)
    token = torch.arange(n, device=x.device).repeat_interleave(k)
    batch = x.new_zeros(e, most, width)
    batch[group[live], place[live]] = x[token[live]]
    h = torch.bmm(batch, _decode_weight(s["w1"][0], s["p1"]).transpose(1, 2)) + s["b1"][:, None, :]
    h = h.clamp_min_(0).view(e * most, -1)
    h = _decode_rows(*_encode_rows(h), h.shape[1]).view(e, most, -1)
    y = torch.bmm(h, _decode_weight(s["w2"][0], s["p2"]).transpose(1, 2)) + s["b2"][:, None, :]
    out = x.new_zeros(n * k, width)
    out[live] = y[group[live], place[live]] * s["weights"].reshape(-1, 1)[live]
    return out.view(n, k, width).sum(dim=1).to(s["x"].dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"route": _route, "quantize": _quantize, "product": _product, "experts": _experts}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# The package's calls
# ---------------------------------------------------------------------------
def _run_own(s):
    from agillm41_b200 import ops

    case = s["case"]
    if case["op"] == "route":
        kw = dict(score=case["score"], renormalize=case["renorm"], scale=case["scale"])
        idx, w = ops.route_experts(s["logits"], case["k"], bias=s["bias"], n_groups=case["groups"],
                                   top_groups=case["keep"], **kw)
        if s["grad"] is None:
            return idx, w
        return idx, w, ops.route_experts_backward(s["grad"], s["logits"], idx, **kw)
    if case["op"] == "quantize":
        t = ops.quantize_fp8(s["x"]) if case["kind"] == "rows" else ops.quantize_fp8_weight(s["x"])
        return ops.dequantize_fp8(t, s["x"].dtype)
    if case["op"] == "product":
        return ops.grouped_gemm_fp8(ops.FP8Tensor(*s["a"]), ops.FP8Tensor(*s["w"]), s["bias"], relu=case["relu"],
                                    seg_start=s["seg_start"], counts=s["counts"], out_dtype=DTYPES[case["dtype"]])
    return ops.moe_experts_fp8(s["x"], s["idx"], s["weights"], ops.FP8Tensor(*s["w1"]), s["b1"],
                               ops.FP8Tensor(*s["w2"]), s["b2"])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if op == "route":
        n, e, k = case["n"], case["e"], case["k"]
        read = n * e * size + (4 * e if case["bias"] else 0)
        written = n * k * 8
        if case["train"]:
            read, written = read + n * k * 4, written + n * e * size
        return {"bytes": read + written, "flops": n * e * (8 if case["train"] else 5)}
    if op == "quantize":
        n = case["g"] * case["n"] * case["width"]
        return {"bytes": n * 2 * size, "flops": 3 * n}
    if op == "product":
        g, rows, n, width = case["g"], case["rows"], case["n"], case["width"]
        used = min(g, rows)
        scales = (rows + used * -(-n // 128)) * -(-width // 128)
        return {"bytes": rows * width + used * n * (width + 4) + rows * n * size + scales, "flops": 2 * rows * n * width}
    n, e, k, width, hidden = (case[x] for x in ("n", "e", "k", "width", "hidden"))
    slots = n * k * (1 - case["drop"])
    used = min(e, max(1, slots))
    return {"bytes": int(2 * n * width * size + n * k * 8 + used * (2 * hidden * width + 4 * (hidden + width))),
            "flops": int(4 * slots * width * hidden)}


# ---------------------------------------------------------------------------
# The operators' definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_e4m3(v):
    """Nearest e4m3 value, ties to even, of |v| <= 448: steps of 2^(e - 3) from the normal range down to 2^-9."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _exact_blocks(x, dims):
    """x with blocks along `dims` -> the values its 8-bit form stands for."""
    amax = x.abs().amax(dim=dims, keepdim=True)
    p = torch.ceil(torch.log2((amax / E4M3_MAX).clamp_min(2.0 ** -127)))
    s = torch.exp2(p)
    return _exact_e4m3(x / s) * s


def _exact_rows(x):
    n, w = x.shape
    wp = -(-w // BLOCK) * BLOCK
    full = x.new_zeros(n, wp)
    full[:, :w] = x
    return _exact_blocks(full.view(n, wp // BLOCK, BLOCK), (2,)).view(n, wp)[:, :w]


def _exact_best(key, k):
    """The k largest of each row, one after the other, the lowest index first among equals."""
    at, found, key = torch.arange(key.shape[1], device=key.device), [], key.clone()
    for _ in range(k):
        best = torch.where(key == key.amax(1, keepdim=True), at, key.shape[1]).amin(1, keepdim=True)
        found.append(best)
        key.scatter_(1, best, -math.inf)
    return torch.cat(found, 1)


def _exact_route(case, s):
    x = s["logits"].double()
    prob = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, 1)
    key = x if s["bias"] is None else prob + s["bias"].double()
    if case["keep"] < case["groups"]:
        parts = (prob if s["bias"] is None else key).unflatten(1, (case["groups"], -1))
        kept = _exact_best(torch.topk(parts, min(2, parts.shape[2]), 2).values.sum(2), case["keep"])
        member = (kept[:, :, None] == torch.arange(case["groups"], device=x.device)).any(1)
        key = key.unflatten(1, (case["groups"], -1)).masked_fill(~member[:, :, None], -math.inf).flatten(1)
    idx = _exact_best(key, case["k"])
    lead = x.gather(1, idx)
    if case["score"] == "sigmoid":
        v = torch.sigmoid(lead)
        t = v / v.sum(1, keepdim=True) if case["renorm"] else v
    elif case["renorm"]:
        v = t = torch.softmax(lead, 1)
    else:
        v = t = torch.exp(lead - torch.logsumexp(x, 1, keepdim=True))
    if s["grad"] is None:
        return idx.to(torch.int32), t * case["scale"]
    leaf = x.clone().requires_grad_(True)
    with torch.enable_grad():
        full = torch.sigmoid(leaf) if case["score"] == "sigmoid" else torch.softmax(leaf, 1)
        c = full.gather(1, idx)
        c = c / c.sum(1, keepdim=True) if case["renorm"] else c
        (c * case["scale"] * s["grad"].double()).sum().backward()
    return idx.to(torch.int32), t * case["scale"], leaf.grad


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(case, s)
    if op == "quantize":
        x = s["x"].double()
        if case["kind"] == "rows":
            return _exact_rows(x)
        g, n, k = x.shape
        full = x.new_zeros(g, -(-n // BLOCK) * BLOCK, -(-k // BLOCK) * BLOCK)
        full[:, :n, :k] = x
        b = full.view(g, full.shape[1] // BLOCK, BLOCK, full.shape[2] // BLOCK, BLOCK)
        return _exact_blocks(b, (2, 4)).view_as(full)[:, :n, :k]

    def values(q, p):
        f = torch.exp2(p.double()).repeat_interleave(BLOCK, -1)
        f = f.repeat_interleave(BLOCK, -2) if q.dim() == 3 else f
        return q.double() * f[..., :q.shape[-2], :q.shape[-1]]

    if op == "product":
        a, w, b = values(s["a"][0], s["ap"]), values(s["w"][0], s["wp"]), s["bias"].double()
        y = a.new_zeros(a.shape[0], case["n"])
        counts = [a.shape[0]] if s["counts"] is None else s["counts"].tolist()
        start = [0] if s["counts"] is None else s["seg_start"].tolist()
        for i, c in enumerate(counts):
            rows = slice(start[i], start[i] + c)
            y[rows] = torch.addmm(b[i], a[rows], w[i].t())
        return torch.relu(y) if case["relu"] else y
    x = _exact_rows(s["x"].double())
    out = torch.zeros_like(x)
    for i in range(case["e"]):
        token, rank = torch.nonzero(s["idx"] == i, as_tuple=True)
        if token.numel():
            h = torch.relu(torch.addmm(s["b1"][i].double(), x[token], values(s["w1"][0][i][None], s["p1"][i][None])[0].t()))
            y = torch.addmm(s["b2"][i].double(), _exact_rows(h), values(s["w2"][0][i][None], s["p2"][i][None])[0].t())
            out.index_add_(0, token, y * s["weights"][token, rank].double()[:, None])
    return out
