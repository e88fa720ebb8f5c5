"""Appending to a paged K/V cache and attention of a batch behind a shared prefix.

Several sequences (continuations of one history, candidates of one step,
single new tokens) keep their own tokens in pages of 64 rows of a resident
cache [1, 64 P, KV heads, 128]; a list of pages that all of them share comes
before their own.  ``append`` rotates new queries and keys by their positions
and writes keys and values to the sequences' next rows; ``attend`` lets each
sequence's new queries see the shared prefix and the sequence's own rows.

Where ``own`` is false, ``run`` computes both with elementary torch
operations in float32 (angles in float64); ``exact`` forms them in float64,
sequence by sequence.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = 'cuda'
D, PAGE = 128, 64
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
VIDEO_AXES = (22, 21, 21)        # pairs that turn with a token's frame, row and column
GRID_H, GRID_W, FRAME = 32, 48, 1536
MOST_FLOPS = 3.2e12              # a drawn call costs no more than the largest listed one
MOST_SCORES = 5.4e9
MOST_ROWS = 8 * 3 * FRAME


def listed():
    return [
        # one new token of one sequence: the smallest append, where latency counts
        dict(name='append_one', kind='append', batch=1, new=1, ragged=False, heads=32, kv_heads=8, held=700, first=0,
             axes=1, pairs=64, interleaved=True, dtype='bf16'),
        # a decode step of 128 sequences far behind a long prefix
        dict(name='append_step_b128', kind='append', batch=128, new=1, ragged=False, heads=32, kv_heads=8, held=2000,
             first=131072, axes=1, pairs=64, interleaved=False, dtype='bf16'),
        # prompts of odd lengths, only the first 80 dims turn
        dict(name='append_ragged', kind='append', batch=24, new=701, ragged=True, heads=28, kv_heads=4, held=300,
             first=5003, axes=1, pairs=40, interleaved=False, dtype='fp16'),
        # a stream's chunk (3 frames) for one layer, keys turned by frame, row and column
        dict(name='append_chunk', kind='append', batch=1, new=4608, ragged=False, heads=12, kv_heads=12, held=0,
             first=15, axes=3, pairs=64, interleaved=True, dtype='bf16'),
        # eight continuations of one history, a chunk each
        dict(name='append_branches', kind='append', batch=8, new=4608, ragged=False, heads=12, kv_heads=12, held=0,
             first=15, axes=3, pairs=64, interleaved=True, dtype='bf16'),
        # one query behind a short prefix of odd length: the smallest call
        dict(name='attend_one', kind='attend', batch=1, new=1, ragged=False, heads=12, kv_heads=12, prefix=1003,
             held=17, causal=True, lse=False, dtype='bf16'),
        # a decode step: 64 sequences behind a common prompt
        dict(name='attend_step_b64', kind='attend', batch=64, new=1, ragged=False, heads=32, kv_heads=8, prefix=16384,
             held=600, causal=True, lse=False, dtype='bf16'),
        # few sequences behind a very long document
        dict(name='attend_long_b16', kind='attend', batch=16, new=1, ragged=False, heads=32, kv_heads=8,
             prefix=131001, held=2100, causal=True, lse=True, dtype='bf16'),
        # five candidate tokens each, checked in one call
        dict(name='attend_verify_b24', kind='attend', batch=24, new=5, ragged=False, heads=28, kv_heads=4, prefix=5003,
             held=333, causal=True, lse=True, dtype='fp16'),
        # prompts of odd lengths after a common one
        dict(name='attend_ragged', kind='attend', batch=6, new=901, ragged=True, heads=32, kv_heads=8, prefix=8192,
             held=1000, causal=True, lse=False, dtype='bf16'),
        # one frame each of eight continuations, behind three frames
        dict(name='attend_frame_b8', kind='attend', batch=8, new=1536, ragged=False, heads=12, kv_heads=12,
             prefix=4608, held=0, causal=False, lse=False, dtype='bf16'),
        # a chunk each of four continuations behind the full history of 360 pages
        dict(name='attend_chunk_b4', kind='attend', batch=4, new=4608, ragged=False, heads=12, kv_heads=12,
             prefix=23040, held=0, causal=False, lse=False, dtype='bf16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kv = rng.choice((1, 2, 3, 4, 8, 12))
    heads = kv * rng.choice((1, 1, 2, 3, 4, 7, 8) if kv < 8 else (1, 1, 2, 4))
    dtype = rng.choice(('bf16', 'bf16', 'fp16'))
    shape = rng.choice(('step', 'step', 'few', 'ragged', 'chunk'))
    batch = _log(rng, 1, 192) if shape == 'step' else _log(rng, 1, 48) if shape == 'few' else _log(rng, 1, 12)
    new = 1 if shape == 'step' else rng.randint(2, 16) if shape == 'few' else _log(rng, 17, 4608)
    new = min(new, MOST_ROWS // batch)
    if rng.random() < 0.4:
        if kv * heads > 144:
            heads = kv
        axes = rng.choice((1, 1, 3))
        return dict(kind='append', batch=batch, new=new, ragged=shape == 'ragged', heads=heads, kv_heads=kv,
                    held=_log(rng, 1, 3000) - 1, first=_log(rng, 1, 200000) - 1, axes=axes,
                    pairs=64 if axes == 3 else rng.choice((64, 64, 32, 48)), interleaved=rng.random() < 0.5,
                    dtype=dtype)
    held = _log(rng, 1, 3000) - 1
    rows = batch * new * heads
    most = min(MOST_FLOPS / (4 * D * rows), MOST_SCORES / rows) - held - new
    prefix = _log(rng, 1, max(1, min(140000, int(most)))) - (rng.random() < 0.1)
    return dict(kind='attend', batch=batch, new=new, ragged=shape == 'ragged', heads=heads, kv_heads=kv,
                prefix=prefix, held=held, causal=rng.random() < 0.7, lse=rng.random() < 0.5, dtype=dtype)


def _counts(case):
    """New tokens of each sequence, and the tokens it holds before them: sizes alone, the same for every seed."""
    B, n, held = case['batch'], case['new'], case['held']
    g = torch.Generator().manual_seed(97 * B + n + held)
    new = torch.full((B,), n)
    if case['ragged']:
        new = torch.randint(0, n + 1, (B,), generator=g)
        new[int(torch.randint(0, B, (1,), generator=g))] = n
    before = torch.randint(0, held + 1, (B,), generator=g)
    before[int(torch.randint(0, B, (1,), generator=g))] = held
    return new, before


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case['dtype']]
    B, H, G = case['batch'], case['heads'], case['kv_heads']
    new, before = _counts(case)
    N = int(new.sum())
    shared = -(-case['prefix'] // PAGE) if case['kind'] == 'attend' else 0
    width = -(-int((new + before).max()) // PAGE)
    pages = shared + B * width
    # pages lie anywhere in the cache, as they do once sequences have come and gone
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    s = dict(case=case, N=N)
    s['prefix'] = order[:shared].contiguous()
    s['table'] = order[shared:].reshape(B, width).contiguous()
    s['starts'] = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32).to(DEV)
    s['most'] = int(new.max())

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dt)

    s['cache_k'], s['cache_v'] = normal(1, PAGE * pages, G, D), normal(1, PAGE * pages, G, D)
    if case['kind'] == 'attend':
        s['q'] = normal(N, H, D)
        s['lengths'] = (before + new).to(torch.int32).to(DEV)
        return s
    # queries, keys and values as one projection leaves them, side by side
    qkv = normal(N, H + 2 * G, D)
    s['q'], s['k'], s['v'] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    s['held'] = before.to(torch.int32).to(DEV)
    R = case['pairs']
    if case['axes'] == 3:
        s['axes'] = VIDEO_AXES
        s['freqs'] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in VIDEO_AXES]).to(DEV)
        i = torch.cat([before[b] + torch.arange(int(new[b])) for b in range(B)])
        frame, cell = i // FRAME + case['first'], i % FRAME
        s['positions'] = torch.stack([frame, cell // GRID_W, cell % GRID_W], 1).to(torch.int32).to(DEV)
    else:
        s['axes'], s['positions'] = (R,), None
        s['freqs'] = (10000.0 ** (-torch.arange(R, dtype=torch.float64) / R)).to(DEV)
    return s


def run(s):
    if own:
        return _own_append(s) if s['case']['kind'] == 'append' else _own_attend(s)
    return _plain_append(s) if s['case']['kind'] == 'append' else _plain_attend(s)


def _own_append(s):
    from streaming_sparse_amd import paged
    from streaming_sparse_amd.attention import Workspace
    c = s['case']
    if 'ws' not in s:
        s['ws'] = Workspace()
    q = paged.append(s['k'], s['v'], s['cache_k'], s['cache_v'], s['table'], s['held'], q=s['q'],
                     starts=s['starts'] if c['ragged'] else None, freqs=s['freqs'], axes=s['axes'],
                     positions=s['positions'], first=c['first'], interleaved=c['interleaved'], workspace=s['ws'])
    return q, s['cache_k'], s['cache_v']


def _own_attend(s):
    from streaming_sparse_amd import paged
    from streaming_sparse_amd.attention import Workspace
    c = s['case']
    if 'ws' not in s:
        s['ws'] = Workspace()
    return paged.attention(s['q'], s['cache_k'], s['cache_v'], s['prefix'], c['prefix'], s['table'], s['lengths'],
                           s['ws'], starts=s['starts'] if c['ragged'] else None, causal=c['causal'],
                           want_lse=c['lse'])


def _sequence_of(s):
    """(sequence, index in it) of every packed row."""
    row = torch.arange(s['N'], device=DEV)
    b = torch.searchsorted(s['starts'][1:].long(), row, right=True)
    return b, row - s['starts'].long()[b]


def _turn(x, cos, sin, interleaved):
    R = cos.shape[-1]
    f = x.float()
    y = f.clone()
    a, b = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if interleaved else (slice(0, R), slice(R, 2 * R))
    y[..., a] = f[..., a] * cos - f[..., b] * sin
    y[..., b] = f[..., a] * sin + f[..., b] * cos
    return y.to(x.dtype)


def _plain_append(s):
    c = s['case']
    b, i = _sequence_of(s)
    at = s['held'].long()[b] + i
    pos = (at + c['first'])[:, None] if s['positions'] is None else s['positions']
    axis = torch.repeat_interleave(torch.arange(len(s['axes']), device=DEV), torch.tensor(s['axes'], device=DEV))
    angle = pos.double()[:, axis] * s['freqs']
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    row = s['table'].long()[b, at // PAGE] * PAGE + at % PAGE
    s['cache_k'][0, row] = _turn(s['k'], cos, sin, c['interleaved'])
    s['cache_v'][0, row] = s['v']
    return _turn(s['q'], cos, sin, c['interleaved']), s['cache_k'], s['cache_v']


def _plain_attend(s):
    c = s['case']
    B, H, G, P, n = c['batch'], c['heads'], c['kv_heads'], c['prefix'], s['most']
    r = H // G
    b, i = _sequence_of(s)
    q = torch.zeros(B, n, H, D, device=DEV)
    q[b, i] = s['q'].float() / math.sqrt(D)
    q = q.reshape(B, n, G, r, D).permute(2, 0, 1, 3, 4)                       # [G, B, n, r, D]

    def pages(x, ids):
        return x[0].reshape(-1, PAGE, G, D)[ids.long()].float()

    kp = pages(s['cache_k'], s['prefix']).reshape(-1, G, D)[:P].permute(1, 2, 0).contiguous()
    vp = pages(s['cache_v'], s['prefix']).reshape(-1, G, D)[:P].permute(1, 0, 2).contiguous()
    ks = pages(s['cache_k'], s['table']).reshape(B, -1, G, D).permute(2, 0, 3, 1).contiguous()
    vs = pages(s['cache_v'], s['table']).reshape(B, -1, G, D).permute(2, 0, 1, 3).contiguous()
    S = vs.shape[2]
    j = torch.arange(S, device=DEV)
    new = s['starts'].long().diff()
    limit = s['lengths'].long()[:, None].expand(B, n)
    if c['causal']:
        limit = torch.minimum(limit, (s['lengths'].long() - new + 1)[:, None] + torch.arange(n, device=DEV))
    hidden = (j >= limit[:, :, None])[None, :, :, None]                       # [1, B, n, 1, S]
    zs = torch.matmul(q.reshape(G, B, n * r, D), ks).reshape(G, B, n, r, S).masked_fill_(hidden, -math.inf)
    top = zs.amax(-1)
    zp = torch.matmul(q.reshape(G, B * n * r, D), kp).reshape(G, B, n, r, P)
    if P:
        top = torch.maximum(top, zp.amax(-1))
    base = top.clamp_min(-3e38)[..., None]
    zs, zp = zs.sub_(base).exp_(), zp.sub_(base).exp_()
    den = zs.sum(-1) + zp.sum(-1)
    o = torch.matmul(zs.reshape(G, B, n * r, S), vs).reshape(G, B, n, r, D)
    o = o + torch.matmul(zp.reshape(G, B * n * r, P), vp).reshape(G, B, n, r, D)
    o = torch.where(den[..., None] > 0, o / den[..., None], 0.0)
    out = o.permute(1, 2, 0, 3, 4).reshape(B, n, H, D)[b, i].to(s['q'].dtype)
    if not c['lse']:
        return out
    return out, (top + den.log()).permute(1, 2, 0, 3).reshape(B, n, H)[b, i]


def work(case):
    new, before = _counts(case)
    new, before = new.double(), before.double()
    N, H, G = float(new.sum()), case['heads'], case['kv_heads']
    if case['kind'] == 'append':
        return dict(bytes=2 * 2 * D * N * (H + 2 * G), flops=3 * 2 * case['pairs'] * N * (H + G))
    held = before + new
    own_keys = new * held
    if case['causal']:
        own_keys = new * before + new * (new + 1) / 2
    keys = float(own_keys.sum()) + N * case['prefix']
    rows = case['prefix'] + float(held.sum())
    return dict(bytes=2 * D * (2 * N * H + 2 * rows * G) + (4 * N * H if case['lse'] else 0), flops=4 * D * H * keys)


def exact(case, seed):
    s = prepare(case, seed)
    lo = s['starts'].tolist()
    H, G = case['heads'], case['kv_heads']
    if case['kind'] == 'append':
        held, table = s['held'].tolist(), s['table'].tolist()
        q, ck, cv = s['q'].double(), s['cache_k'].double(), s['cache_v'].double()
        which = [a for a, n in enumerate(s['axes']) for _ in range(n)]
        R = len(which)
        first, second = (torch.arange(R) * 2, torch.arange(R) * 2 + 1) if case['interleaved'] else \
            (torch.arange(R), torch.arange(R) + R)
        for b in range(case['batch']):
            n = lo[b + 1] - lo[b]
            if n == 0:
                continue
            at = held[b] + torch.arange(n, device=DEV, dtype=torch.float64)
            pos = (at + case['first'])[:, None] if s['positions'] is None else s['positions'][lo[b]:lo[b + 1]].double()
            z = torch.polar(torch.ones(n, R, dtype=torch.float64, device=DEV), pos[:, which] * s['freqs'])[:, None]

            def turned(x):
                w = torch.complex(x[..., first.to(DEV)], x[..., second.to(DEV)]) * z
                y = x.clone()
                y[..., first.to(DEV)], y[..., second.to(DEV)] = w.real, w.imag
                return y

            rows = torch.tensor([PAGE * table[b][(held[b] + i) // PAGE] + (held[b] + i) % PAGE for i in range(n)],
                                device=DEV)
            q[lo[b]:lo[b + 1]] = turned(q[lo[b]:lo[b + 1]])
            ck[0, rows] = turned(s['k'][lo[b]:lo[b + 1]].double())
            cv[0, rows] = s['v'][lo[b]:lo[b + 1]].double()
        return q, ck, cv
    if case['batch'] * G > 600:
        return None
    out = torch.zeros(s['N'], H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((s['N'], H), -math.inf, dtype=torch.float64, device=DEV)
    length, P = s['lengths'].tolist(), case['prefix']
    flat_k, flat_v = s['cache_k'][0].view(-1, PAGE, G, D), s['cache_v'][0].view(-1, PAGE, G, D)
    for b in range(case['batch']):
        n, own_pages = lo[b + 1] - lo[b], -(-length[b] // PAGE)
        if n == 0:
            continue
        for h in range(G):
            def rows(flat):
                return torch.cat([flat[s['prefix'].long(), :, h].reshape(-1, D)[:P],
                                  flat[s['table'][b, :own_pages].long(), :, h].reshape(-1, D)[:length[b]]]).double()

            k, v = rows(flat_k), rows(flat_v)
            seen = P + (length[b] - n + torch.arange(n, device=DEV) + 1 if case['causal'] else
                        torch.full((n,), length[b], device=DEV))
            for hq in range(h * (H // G), (h + 1) * (H // G)):
                z = s['q'][lo[b]:lo[b + 1], hq].double() @ k.t() * D ** -0.5
                z = z.masked_fill(torch.arange(P + length[b], device=DEV) >= seen[:, None], -math.inf)
                lse[lo[b]:lo[b + 1], hq] = torch.logsumexp(z, -1)
                out[lo[b]:lo[b + 1], hq] = torch.softmax(z, -1).nan_to_num(0.0) @ v
    return (out, lse) if case['lse'] else out
