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



def error_limit(want, p2, p2v2, dtype, parts, part=None):
    """What the root of the summed squared errors of outputs `want` [..., 128] may
    be, given sum p^2 [...] and sum p^2 v^2 [..., 128] over their normalised
    probabilities, each of which meets V in `parts` 16-bit parts, one of which is of
    type `part` (else of the outputs').

    * A result rounded once is off by an error uniform within half a step: mean
      square step^2 / 12, the sum's standard deviation sqrt(4 / 5) of the root of
      the squared means' sum.  Six of those are allowed, here and below.
    * One part: a probability is off by at most eps / 2 of itself (the part's), mean square
      below eps^2 / 12, one error for all 128 dims: their quadratic form over a row
      has the mean eps^2 / 12 sum p^2 v^2 and a variance of at most twice its square
      times 1 / 128 + sum p^2.
    * The rest, as a part of each probability and of the output: scores' 128
      float32 roundings of sums below 16 (root mean square 2^-18), exponents
      and exponentials (2^-20), a second part's rounding (below 2^-16 in bf16, 2^-22
      in fp16), sums of up to 2^15 terms (2^-17): 2^-15.
    Errors of different origin add up as their roots at most."""
    info = torch.finfo(dtype)
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(info.smallest_normal)))) * info.eps
    e = step * step / 12
    limit = (e.sum() + 6 * (0.8 * (e * e).sum()).sqrt()).sqrt()
    if parts == 1:
        e = p2v2.sum(-1) * torch.finfo(part or dtype).eps ** 2 / 12
        limit = limit + (e.sum() + 6 * (2 * (e * e * (1 / 128 + p2)).sum()).sqrt()).sqrt()
    return limit + 2.0 ** -15 * (p2v2.sum() + (want * want).sum()).sqrt()
