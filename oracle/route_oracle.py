"""General expert routing from its definition, in 64 bits (test infrastructure only)."""
import math

import torch


def scores(l, score):
    if score == "sigmoid":
        return torch.sigmoid(l)
    m = l.amax(dim=1, keepdim=True)
    z = torch.exp(l - torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m))
    z = torch.where((l == m) & (m > 0) & torch.isinf(m), torch.ones_like(z), z)   # beside +inf: the limit
    return z / z.sum(dim=1, keepdim=True).clamp_min(1e-300)


def _best(key, k):
    """Indices of the k largest, lowest first among equals; -1 where only -inf is left."""
    key = key.clone()
    at = torch.arange(key.shape[1], device=key.device)
    out = []
    for _ in range(k):
        top = key.amax(1, keepdim=True)
        i = torch.where(key == top, at, key.shape[1]).amin(1, keepdim=True)
        out.append(torch.where(top > -math.inf, i, torch.full_like(i, -1)))
        key.scatter_(1, i, -math.inf)
    return torch.cat(out, 1)


def choose(logits, k, score="softmax", bias=None, n_groups=1, top_groups=None):
    l = logits.double()
    s = scores(torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l), score)
    key = l if bias is None else s + bias.double()
    off = torch.isnan(key) | torch.isnan(l) | (l == -math.inf)
    key = key.masked_fill(off, -math.inf)
    top_groups = n_groups if top_groups is None else top_groups
    if top_groups < n_groups:
        n, E = l.shape
        part = (s if bias is None else key).masked_fill(key == -math.inf, -math.inf).view(n, n_groups, -1)
        two = part.topk(min(2, part.shape[2]), dim=2).values
        g = two[..., 0].clone()
        if two.shape[2] == 2:
            g = torch.where(two[..., 1] > -math.inf, two.sum(2), g)
        kept = _best(g, top_groups)
        member = (kept[:, :, None] == torch.arange(n_groups, device=l.device)).any(1)
        key = key.view(n, n_groups, -1).masked_fill(~member[:, :, None], -math.inf).view(n, E)
    return _best(key, k)


def weights(logits, idx, score="softmax", renormalize=True, scale=1.0):
    """[N, k] float64, differentiable in the logits; empty slots 0."""
    l = logits.double()
    live = idx >= 0
    at = idx.clamp_min(0).long()
    c = l.gather(1, at)
    if renormalize:
        # ratios of scores, from their logarithms: they stay exact where every score underflows
        log = c if score == "softmax" else torch.nn.functional.logsigmoid(c)
        w = torch.softmax(log.masked_fill(~live, -math.inf), 1)
    elif score == "softmax":
        w = torch.softmax(l, 1).gather(1, at)   # exp(l - logsumexp) would lose the sum beside logits of -3.4e38
    else:
        w = torch.sigmoid(c)
    return torch.where(live, w, torch.zeros_like(w)) * scale
