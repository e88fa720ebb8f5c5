"""float64 restatement of the paged append and the shared-prefix attention,
sequence by sequence on the CPU."""
from __future__ import annotations

import math

import torch

PAGE = 64


def rotate(x, positions, freqs, axes, interleaved):
    """x [n, heads, 128] float64 turned by positions [n, A] (int64)."""
    R = freqs.numel()
    axis = [a for a, n in enumerate(axes) for _ in range(n)]
    angle = positions.double()[:, axis] * freqs.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    first = torch.arange(0, 2 * R, 2) if interleaved else torch.arange(R)
    second = first + (1 if interleaved else R)
    y = x.clone()
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., first] * sin + x[..., second] * cos
    return y


def append(k, v, cache_k, cache_v, table, held, starts, q=None, freqs=None, axes=None, positions=None, first=0,
           interleaved=True):
    """(q rotated or None, cache_k, cache_v, touched rows): float64 copies on
    the CPU with the new tokens written."""
    k, v, table = k.cpu().double(), v.cpu().double(), table.cpu()
    ck, cv = cache_k[0].cpu().double().clone(), cache_v[0].cpu().double().clone()
    q = None if q is None else q.cpu().double().clone()
    starts, held = starts.tolist(), held.tolist()
    touched = torch.zeros(ck.shape[0], dtype=torch.bool)
    for b in range(len(held)):
        lo, hi = starts[b], starts[b + 1]
        at = held[b] + torch.arange(hi - lo)
        if freqs is not None and hi > lo:
            pos = (at + first)[:, None] if positions is None else positions.cpu()[lo:hi].reshape(hi - lo, -1)
            ax = axes or (freqs.numel(),)
            turned = rotate(k[lo:hi], pos, freqs.cpu(), ax, interleaved)
            if q is not None:
                q[lo:hi] = rotate(q[lo:hi], pos, freqs.cpu(), ax, interleaved)
        else:
            turned = k[lo:hi]
        for i, a in enumerate(at.tolist()):
            if not 0 <= a < PAGE * table.shape[1]:
                continue
            page = int(table[b, a // PAGE])
            if not 0 <= page < ck.shape[0] // PAGE:
                continue
            row = PAGE * page + a % PAGE
            ck[row], cv[row], touched[row] = turned[i], v[lo + i], True
    return q, ck[None], cv[None], touched


def attention(q, cache_k, cache_v, prefix, prefix_tokens, table, lengths, starts, causal=True, scale=None):
    """(out, lse, spread) float64: spread is sum p |v| / sum p, the size that a
    relative error of the probabilities is measured by.  Rows behind the last
    sequence are NaN."""
    q, ck, cv, table = q.cpu().double(), cache_k[0].cpu(), cache_v[0].cpu(), table.cpu()
    n_all, H, D = q.shape
    G = ck.shape[1]
    P = ck.shape[0] // PAGE
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((n_all, H, D), math.nan, dtype=torch.float64)
    spread, lse = out.clone(), torch.full((n_all, H), math.nan, dtype=torch.float64)
    starts, lengths = starts.tolist(), lengths.tolist()
    shared = [] if prefix is None else prefix.tolist()

    def rows(pages, count):
        # cache rows, -1 where a page is absent; none of those behind the list
        got, count = [], min(count, PAGE * len(pages))
        for i in range(-(-count // PAGE)):
            if 0 <= pages[i] < P:
                got += [PAGE * pages[i] + r for r in range(min(PAGE, count - PAGE * i))]
            else:
                got += [-1] * min(PAGE, count - PAGE * i)
        return torch.tensor(got, dtype=torch.long)

    pre = rows(shared, prefix_tokens)
    for b, length in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        own = rows(table[b].tolist(), length)
        for t in range(lo, hi):
            last = min(length, length - (hi - lo) + (t - lo) + 1) if causal else length
            at = torch.cat([pre, own[:max(last, 0)]])
            at = at[at >= 0]
            for h in range(H):
                kk, vv = ck[at, h // (H // G)].double(), cv[at, h // (H // G)].double()
                z = kk @ q[t, h] * scale
                lse[t, h] = torch.logsumexp(z, 0) if len(at) else -math.inf
                p = torch.softmax(z, 0)
                out[t, h] = p @ vv if len(at) else 0.0
                spread[t, h] = p @ vv.abs() if len(at) else 0.0
    return out, lse, spread
