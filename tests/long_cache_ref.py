"""Plain float64 forms of the operators for long caches, on the CPU, written from
their definitions one token and one page at a time."""

import math

import torch

import serving_ref as R


def bounds(keys, d, dp):
    """[2, dp]: least and largest value of each column of the keys [tokens, d] a page holds."""
    out = torch.zeros(2, dp)
    out[0, :d] = keys.amin(0).float()
    out[1, :d] = keys.amax(0).float()
    return out.to(torch.bfloat16)


def _order(x):
    """Sorts the largest first, NaN before all."""
    return (0, 0.0) if math.isnan(x) else (1, -x)


def select(q, low, high, pages, count, first, last):
    """Rows of the table for one query token and key head: q [group, d], low / high [W, d]
    float64; of rows 0 .. pages - 1."""
    if pages <= count:
        return list(range(pages)) + [-1] * (count - pages)
    fixed = list(range(first)) + list(range(pages - last, pages))
    scores = {}
    for w in range(first, pages - last):
        scores[w] = _order(torch.maximum(q * low[w], q * high[w]).sum().item())
    best = sorted(scores, key=lambda w: (scores[w], w))[:count - first - last]
    return sorted(fixed + best)


def keep_of(weights, keep, first, last):
    """Tokens that stay, of one request and head: weights [tokens]."""
    n = len(weights)
    fixed = list(range(first)) + list(range(n - last, n))
    value = {j: _order(weights[j]) for j in range(first, n - last)}
    best = sorted(value, key=lambda j: (value[j], j))[:keep - first - last]
    return sorted(fixed + best)


def attend(q, k, v, sees, scale):
    """q [n, heads, d], k / v [m, kv heads, d] float64, sees [n, m] or [kv heads, n, m]: out [n, heads, d], the
    magnitudes that errors scale with (serving_ref.attention), and p [heads, n, m]."""
    heads, h = q.shape[1], k.shape[1]
    per = heads // h
    sees = sees if sees.ndim == 3 else sees.expand(h, -1, -1)
    outs, spreads, scores, ps = [], [], [], []
    for i in range(h):
        qi, ki, vi = q[:, i * per:(i + 1) * per].transpose(0, 1), k[:, i].expand(per, -1, -1), v[:, i].expand(per, -1, -1)
        o, spread, score = R.attention(qi, ki, vi, sees[i], scale)
        x = torch.einsum("hnd,hmd->hnm", qi, torch.where(sees[i].any(0)[None, :, None], ki, torch.zeros_like(ki))) * scale
        x = torch.where(sees[i], x, torch.full((), -math.inf, dtype=torch.float64))
        ps.append(torch.nan_to_num(torch.softmax(x, -1), nan=0.0))
        outs.append(o)
        spreads.append(spread)
        scores.append(score)
    return tuple(torch.cat(t).transpose(0, 1) for t in (outs, spreads, scores)) + (torch.cat(ps),)
