"""float64 restatement of the 8-bit paged cache and of attention with shaped
scores, sequence by sequence on the tensors' own device."""
from __future__ import annotations

import math

import torch

PAGE = 64


def exponents(x):
    """Biased exponents of 16-bit rows [..., 128]: the smallest from 1 on with which a row's largest finite magnitude
    stays within 448."""
    top = torch.where(torch.isfinite(x), x, 0).double().abs().amax(-1)
    s = torch.full(top.shape, 1, dtype=torch.long, device=x.device)
    for e in range(2, 255):
        s = torch.where(top > 448 * 2.0 ** (e - 1 - 127), e, s)
    return s


def quantise(x, s=None):
    """(values, biased exponents) of 16-bit rows [..., 128]: float64 values on the e4m3
    grid, which times 2^(s - 127) are what the rows stand for."""
    s = exponents(x) if s is None else s
    y, finite = x.double(), torch.isfinite(x)
    # rounded up, these would be infinite in their 16-bit type
    last = 2.0 ** (15 if x.dtype is torch.float16 else 127)
    y = torch.where(y.abs() >= 1.9375 * last, torch.copysign(torch.full_like(y, 1.875 * last), y), y)
    y = torch.where(finite, y, 0.0) * torch.exp2((127 - s).double())[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    y = torch.round(y / step) * step    # half to even
    return torch.where(finite, y, math.nan), s


def values(x8, s):
    """float64 values that e4m3 values [..., 128] with their rows' exponents stand for."""
    return x8.double() * torch.exp2(s.double() - 127)[..., None]


def pages16(cache):
    """[P, G, 64, 128] float64 of a 16-bit cache [1, 64 P, G, 128]."""
    return cache[0].unflatten(0, (-1, PAGE)).transpose(1, 2).double()


def pages8(cache):
    return values(cache.k, cache.scales[:, :, 0]), values(cache.v, cache.scales[:, :, 1])


def attention(q, k, v, prefix, prefix_tokens, table, lengths, starts, causal=True, scale=None, cap=None, slopes=None,
              window=None):
    """(out, lse, spread) float64 of pages [P, G, 64, 128]: spread is sum p |v| / sum p.
    Rows behind the last sequence are NaN."""
    n_all, H, D = q.shape
    P, G = k.shape[:2]
    dev = q.device
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((n_all, H, D), math.nan, dtype=torch.float64, device=dev)
    spread, lse = out.clone(), torch.full((n_all, H), math.nan, dtype=torch.float64, device=dev)

    def rows(ids, count):
        """(cache page or -1, row in it, place) of the rows of a list."""
        i = torch.arange(min(count, PAGE * len(ids)), device=dev)
        page = ids.long().to(dev)[i // PAGE]
        return torch.where((page >= 0) & (page < P), page, -1), i % PAGE, i

    none = torch.zeros(0, dtype=torch.int32, device=dev)
    pre = rows(none if prefix is None else prefix, prefix_tokens)
    starts, lengths = starts.tolist(), lengths.tolist()
    for b, length in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        if n == 0:
            continue
        own = rows(table[b], length)
        page, row = (torch.cat([x, y]) for x, y in zip(pre[:2], own[:2]))
        place = torch.cat([pre[2], own[2] + prefix_tokens])
        mine = torch.cat([torch.zeros_like(pre[2], dtype=torch.bool), torch.ones_like(own[2], dtype=torch.bool)])
        at = prefix_tokens + length - n + torch.arange(n, device=dev)[:, None]      # the queries' own places
        hidden = (page < 0).expand(n, -1)
        if causal:
            hidden = hidden | mine & (place > at)
        if window is not None:
            hidden = hidden | mine & (place <= at - window)
        seen = ~hidden.all(0)
        page, row, place, hidden = page[seen], row[seen], place[seen], hidden[:, seen]
        part = slice(starts[b], starts[b + 1])
        for g in range(G):
            kk, vv = k[page, g, row], v[page, g, row]
            for h in range(g * (H // G), (g + 1) * (H // G)):
                z = q[part, h].double() @ kk.t() * scale
                if cap is not None:
                    z = cap * torch.tanh(z / cap)
                if slopes is not None:
                    z = z - slopes[h].double() * (at - place).abs()
                z = z.masked_fill(hidden, -math.inf)
                p = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e300)) if len(place) else z
                total = p.sum(-1, keepdim=True)
                p = torch.where(total > 0, p / total, 0.0)
                out[part, h], spread[part, h] = p @ vv, p @ vv.abs()
                lse[part, h] = torch.logsumexp(z, -1) if len(place) else -math.inf
    return out, lse, spread
