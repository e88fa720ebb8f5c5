"""An 8-bit paged K/V cache (written, read back, attended), and attention whose
scores are capped, fall with distance or see a sliding window.

The 8-bit cache holds a row of 128 elements of one head as e4m3 values and one
power of two: pages [P, G, 64, 128] of keys and of values, scales [P, G, 2, 64]
(keys', then values') as biased exponents (2^(s - 127)).  Several sequences own
pages through a table, as in the 16-bit cache [1, 64 P, G, 128]; a list of
pages that all share comes before their own.

* write: new queries and keys are rotated by their positions, keys and values
  quantised into the sequences' next rows, and those rows read back as the
  values that later steps will see;
* read: rows of several sequences from the 8-bit cache, packed, in 16 bits;
* attend: new queries over the shared prefix and their sequence's own rows, of
  the 8-bit cache (`bits` 8) or the 16-bit one (16).  A score is scale q.k;
  with `cap` it becomes cap tanh(score / cap), with `slopes` it falls by a head's
  slope times the distance in tokens, with `window` a query sees only the
  `window` rows of its own sequence up to itself (and the whole prefix).

Where ``own`` is false, ``run`` computes them with elementary torch operations
in float32 (rotations in float64, next to a rounding's border); ``exact`` forms
them in float64, sequence by sequence.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = 'cuda'
D, PAGE = 128, 64
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
VIDEO_AXES = (22, 21, 21)        # pairs that turn with a token's frame, row and column
GRID_W, FRAME = 48, 1536
MOST_FLOPS = 3.2e12              # a drawn call costs no more than the largest listed one
MOST_SCORES = 5.4e9
MOST_ROWS = 8 * 3 * FRAME
MOST_HELD = 4.6e6                # rows times heads of the sequences' own pages


def listed():
    return [
        # one new token of one sequence: the smallest write, where latency counts
        dict(name='write_one', kind='write', batch=1, new=1, ragged=False, heads=32, kv_heads=8, held=700, first=0,
             axes=1, pairs=64, interleaved=True, dtype='bf16'),
        # prompts of odd lengths, only the first 80 dims turn
        dict(name='write_ragged', kind='write', batch=24, new=701, ragged=True, heads=28, kv_heads=4, held=300,
             first=5003, axes=1, pairs=40, interleaved=False, dtype='fp16'),
        # eight continuations of one history, a chunk (3 frames) each, keys turned by frame, row and column
        dict(name='write_branches', kind='write', batch=8, new=4608, ragged=False, heads=12, kv_heads=12, held=0,
             first=15, axes=3, pairs=64, interleaved=True, dtype='bf16'),
        # odd runs of rows of many sequences, handed back in 16 bits
        dict(name='read_ragged', kind='read', batch=40, new=331, ragged=True, heads=4, kv_heads=4, held=900,
             dtype='fp16'),
        # one continuation's history of 360 pages back into a 16-bit window
        dict(name='read_history', kind='read', batch=1, new=23040, ragged=False, heads=12, kv_heads=12, held=0,
             dtype='bf16'),
        # one query behind a short prefix of odd length: the smallest call
        dict(name='attend_one', kind='attend', bits=8, batch=1, new=1, ragged=False, heads=12, kv_heads=12, prefix=1003,
             held=17, causal=True, lse=False, cap=0.0, slopes=False, window=0, dtype='bf16'),
        # a decode step: 64 sequences behind a common prompt
        dict(name='attend_step_b64', kind='attend', bits=8, batch=64, new=1, ragged=False, heads=32, kv_heads=8,
             prefix=16384, held=600, causal=True, lse=False, cap=0.0, slopes=False, window=0, dtype='bf16'),
        # few sequences behind a very long document
        dict(name='attend_long_b16', kind='attend', bits=8, batch=16, new=1, ragged=False, heads=32, kv_heads=8,
             prefix=131001, held=2100, causal=True, lse=True, cap=0.0, slopes=False, window=0, dtype='bf16'),
        # a chunk each of four continuations behind the full history of 360 pages
        dict(name='attend_chunk_b4', kind='attend', bits=8, batch=4, new=4608, ragged=False, heads=12, kv_heads=12,
             prefix=23040, held=0, causal=False, lse=False, cap=0.0, slopes=False, window=0, dtype='bf16'),
        # a decode step of long sequences behind a few fixed first rows, capped scores, pages behind the window released
        dict(name='shaped_step_b48', kind='attend', bits=8, batch=48, new=1, ragged=False, heads=32, kv_heads=8,
             prefix=64, held=12000, causal=True, lse=False, cap=30.0, slopes=False, window=4096, dtype='bf16'),
        # five candidate tokens each, checked in one call; scores fall with distance
        dict(name='shaped_verify_b24', kind='attend', bits=16, batch=24, new=5, ragged=False, heads=28, kv_heads=4,
             prefix=5003, held=333, causal=True, lse=True, cap=0.0, slopes=True, window=0, dtype='fp16'),
        # prompts of odd lengths continued in a window, capped
        dict(name='shaped_ragged', kind='attend', bits=16, batch=6, new=1801, ragged=True, heads=32, kv_heads=8,
             prefix=64, held=6000, causal=True, lse=False, cap=50.0, slopes=False, window=2048, dtype='bf16'),
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
    kind = rng.choice(('write', 'read', 'attend', 'attend', 'shaped', 'shaped'))
    if kind == 'read':
        return dict(kind='read', batch=batch, new=_log(rng, 1, min(23040, MOST_ROWS // batch)), ragged=rng.random() < 0.6,
                    heads=kv, kv_heads=kv, held=_log(rng, 1, 3000) - 1, dtype=dtype)
    if kind == 'write':
        if kv * heads > 144:
            heads = kv
        axes = rng.choice((1, 1, 3))
        return dict(kind='write', batch=batch, new=new, ragged=shape == 'ragged', heads=heads, kv_heads=kv,
                    held=_log(rng, 1, 3000) - 1, first=_log(rng, 1, 200000) - 1, axes=axes,
                    pairs=64 if axes == 3 else rng.choice((64, 64, 32, 48)), interleaved=rng.random() < 0.5,
                    dtype=dtype)
    new = min(new, int(math.sqrt(MOST_SCORES / (batch * heads))))
    rows = batch * new * heads
    most = min(MOST_FLOPS / (4 * D * rows), MOST_SCORES / rows) - new
    shaped = kind == 'shaped'
    held = _log(rng, 1, max(1, int(min(20000 if shaped else 3000, MOST_HELD / (batch * kv), most / 2)))) - 1
    prefix = _log(rng, 1, max(1, min(8000 if shaped else 140000, int(most - held)))) - (rng.random() < 0.1)
    cap, slopes, window = 0.0, False, 0
    if shaped:
        how = rng.choice(('cap', 'slopes', 'window', 'cap and window', 'all'))
        cap = float(rng.choice((5, 20, 30, 50))) if how in ('cap', 'cap and window', 'all') else 0.0
        slopes = how in ('slopes', 'all')
        window = _log(rng, 16, 8192) if how in ('window', 'cap and window', 'all') else 0
    return dict(kind='attend', bits=rng.choice((8, 16)) if shaped else 8, batch=batch, new=new, ragged=shape == 'ragged',
                heads=heads, kv_heads=kv, prefix=prefix, held=held, causal=rng.random() < 0.7, lse=rng.random() < 0.5,
                cap=cap, slopes=slopes, window=window, dtype=dtype)


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


def _quantised(x):
    """e4m3 values and biased exponents (uint8) of rows [..., 128]: the smallest power of two with which the row's
    largest magnitude stays within 448."""
    top = x.abs().amax(-1).double()
    m, e = torch.frexp(top)                                  # top = m 2^e, 0.5 <= m < 1
    s = (e + 127 - 9 + (m > 0.875)).clamp(1, 254)            # 448 = 0.875 * 2^9
    return (x * torch.exp2((127 - s).to(x.dtype))[..., None]).to(torch.float8_e4m3fn), s.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case['dtype']]
    B, H, G, kind = case['batch'], case['heads'], case['kv_heads'], case['kind']
    new, before = _counts(case)
    N = int(new.sum())
    shared = -(-case['prefix'] // PAGE) if kind == 'attend' else 0
    width = -(-int((new + before).max()) // PAGE)
    pages = shared + B * width
    # pages lie anywhere in the cache, as they do once sequences have come and gone
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    s = dict(case=case, N=N)
    s['prefix'] = order[:shared].contiguous()
    s['table'] = order[shared:].reshape(B, width).contiguous()
    s['starts'] = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32).to(DEV)
    s['held'] = before.to(torch.int32).to(DEV)
    s['most'] = int(new.max())

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    if kind == 'write':
        s['k8'], s['v8'] = (torch.zeros(pages, G, PAGE, D, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
        s['scales'] = torch.full((pages, G, 2, PAGE), 127, device=DEV, dtype=torch.uint8)
    elif kind == 'read' or case['bits'] == 8:
        # heads differ in size, and a row in eight is much smaller than the others
        gain = torch.exp2(torch.randint(-3, 4, (1, G, 1, 1), generator=g, device=DEV).float())
        small = torch.where(torch.rand(pages, G, PAGE, 1, generator=g, device=DEV) < 0.125, 2.0 ** -6, 1.0)
        s['k8'], sk = _quantised(normal(pages, G, PAGE, D))
        s['v8'], sv = _quantised(normal(pages, G, PAGE, D) * gain * small)
        s['scales'] = torch.stack([sk, sv], 2).contiguous()
    else:
        s['cache_k'], s['cache_v'] = normal(1, PAGE * pages, G, D).to(dt), normal(1, PAGE * pages, G, D).to(dt)
    if kind == 'read':
        return s
    if kind == 'attend':
        s['q'] = normal(N, H, D).to(dt)
        s['lengths'] = (before + new).to(torch.int32).to(DEV)
        s['slopes'] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H) if case['slopes'] else None
        if case['window']:
            # pages that have fallen out of every query's window are released
            gone = (before - case['window'] + 1).clamp_min(0) // PAGE
            s['table'][torch.arange(width)[None] < gone[:, None]] = -1
        return s
    # queries, keys and values as one projection leaves them, side by side
    qkv = normal(N, H + 2 * G, D).to(dt)
    s['q'], s['k'], s['v'] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
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
    kind = s['case']['kind']
    if own:
        return _own_write(s) if kind == 'write' else _own_read(s) if kind == 'read' else _own_attend(s)
    return _plain_write(s) if kind == 'write' else _plain_read(s) if kind == 'read' else _plain_attend(s)


def _own_state(s):
    from streaming_sparse_amd import paged8
    from streaming_sparse_amd.attention import Workspace
    s['ws'] = Workspace()
    if 'k8' in s:
        s['cache'] = paged8.Cache(s['k8'], s['v8'], s['scales'])


def _own_write(s):
    from streaming_sparse_amd import paged8
    c = s['case']
    if 'ws' not in s:
        _own_state(s)
    starts = s['starts'] if c['ragged'] else None
    q = paged8.append(s['k'], s['v'], s['cache'], s['table'], s['held'], q=s['q'], starts=starts, freqs=s['freqs'],
                      axes=s['axes'], positions=s['positions'], first=c['first'], interleaved=c['interleaved'],
                      workspace=s['ws'])
    k, v = paged8.read(s['cache'], s['table'], s['held'], s['N'], starts=starts, dtype=s['k'].dtype,
                       workspace=s['ws'])
    return q, k, v


def _own_read(s):
    from streaming_sparse_amd import paged8
    c = s['case']
    if 'ws' not in s:
        _own_state(s)
    return paged8.read(s['cache'], s['table'], s['held'], s['N'], starts=s['starts'] if c['ragged'] else None,
                       dtype=TYPES[c['dtype']], workspace=s['ws'])


def _own_attend(s):
    from streaming_sparse_amd import paged, paged8
    c = s['case']
    if 'ws' not in s:
        _own_state(s)
    more = dict(starts=s['starts'] if c['ragged'] else None, causal=c['causal'], want_lse=c['lse'],
                cap=c['cap'] or None, slopes=s['slopes'], window=c['window'] or None)
    if c['bits'] == 8:
        return paged8.attention(s['q'], s['cache'], s['prefix'], c['prefix'], s['table'], s['lengths'], s['ws'], **more)
    return paged.attention(s['q'], s['cache_k'], s['cache_v'], s['prefix'], c['prefix'], s['table'], s['lengths'],
                           s['ws'], **more)


def _sequence_of(s):
    """(sequence, index in it) of every packed row."""
    row = torch.arange(s['N'], device=DEV)
    b = torch.searchsorted(s['starts'][1:].long(), row, right=True)
    return b, row - s['starts'].long()[b]


def _turn(x, cos, sin, interleaved):
    R = cos.shape[-1]
    f = x.double()
    y = f.clone()
    a, b = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if interleaved else (slice(0, R), slice(R, 2 * R))
    y[..., a] = f[..., a] * cos - f[..., b] * sin
    y[..., b] = f[..., a] * sin + f[..., b] * cos
    return y.to(x.dtype)


def _values(x8, scale):
    return x8.float() * torch.exp2(scale.float() - 127.0)[..., None]


def _plain_write(s):
    c = s['case']
    b, i = _sequence_of(s)
    at = s['held'].long()[b] + i
    pos = (at + c['first'])[:, None] if s['positions'] is None else s['positions']
    axis = torch.repeat_interleave(torch.arange(len(s['axes']), device=DEV), torch.tensor(s['axes'], device=DEV))
    angle = pos.double()[:, axis] * s['freqs']
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    page, row = s['table'].long()[b, at // PAGE], at % PAGE
    k8, sk = _quantised(_turn(s['k'], cos, sin, c['interleaved']).float())
    v8, sv = _quantised(s['v'].float())
    s['k8'].view(torch.uint8)[page, :, row] = k8.view(torch.uint8)
    s['v8'].view(torch.uint8)[page, :, row] = v8.view(torch.uint8)
    s['scales'][page, :, 0, row], s['scales'][page, :, 1, row] = sk, sv
    return (_turn(s['q'], cos, sin, c['interleaved']), *_plain_read(s))


def _plain_read(s):
    b, i = _sequence_of(s)
    at = s['held'].long()[b] + i
    page, row, dt = s['table'].long()[b, at // PAGE], at % PAGE, TYPES[s['case']['dtype']]
    k8, v8 = (s[x].view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn) for x in ('k8', 'v8'))
    scale = s['scales'][page, :, :, row]
    return _values(k8, scale[..., 0]).to(dt), _values(v8, scale[..., 1]).to(dt)


def _pages(s, ids):
    """Keys and values [..., G, 64, 128] float32 of pages `ids` (those released read page 0)."""
    ids = ids.long().clamp_min(0)
    if s['case']['bits'] == 8:
        scale = s['scales'][ids]
        return (_values(s[x].view(torch.uint8)[ids].view(torch.float8_e4m3fn), scale[..., i, :])
                for i, x in enumerate(('k8', 'v8')))
    G = s['case']['kv_heads']
    return (s[x][0].reshape(-1, PAGE, G, D)[ids].float().transpose(-3, -2) for x in ('cache_k', 'cache_v'))


def _shape(z, c, slopes, distance):
    """z [G, B, n, r, keys] in place, distance [B, n, keys]."""
    if c['cap']:
        z.div_(c['cap']).tanh_().mul_(c['cap'])
    if slopes is not None:
        G, r = z.shape[0], z.shape[3]
        z.addcmul_(slopes.view(G, 1, 1, r, 1), distance.abs()[None, :, :, None].float(), value=-1.0)
    return z


def _plain_attend(s):
    c = s['case']
    B, H, G, P, n = c['batch'], c['heads'], c['kv_heads'], c['prefix'], s['most']
    r = H // G
    b, i = _sequence_of(s)
    q = torch.zeros(B, n, H, D, device=DEV)
    q[b, i] = s['q'].float() / math.sqrt(D)
    q = q.reshape(B, n, G, r, D).permute(2, 0, 1, 3, 4)                       # [G, B, n, r, D]
    kp, vp = _pages(s, s['prefix'])                                           # [pages, G, 64, D]
    kp = kp.transpose(0, 1).reshape(G, -1, D)[:, :P].transpose(1, 2).contiguous()
    vp = vp.transpose(0, 1).reshape(G, -1, D)[:, :P].contiguous()
    ks, vs = _pages(s, s['table'])                                            # [B, pages, G, 64, D]
    ks = ks.permute(2, 0, 4, 1, 3).reshape(G, B, D, -1).contiguous()
    vs = vs.permute(2, 0, 1, 3, 4).reshape(G, B, -1, D).contiguous()
    S = vs.shape[2]
    j = torch.arange(S, device=DEV)
    new = s['starts'].long().diff()
    at = (s['lengths'].long() - new)[:, None] + torch.arange(n, device=DEV)   # a query's own row
    limit = s['lengths'].long()[:, None].expand(B, n)
    if c['causal']:
        limit = torch.minimum(limit, at + 1)
    hidden = j >= limit[:, :, None]
    if c['window']:
        hidden |= j <= (at - c['window'])[:, :, None]
    zs = torch.matmul(q.reshape(G, B, n * r, D), ks).reshape(G, B, n, r, S)
    zs = _shape(zs, c, s['slopes'], at[:, :, None] - j if c['slopes'] else None)
    zs.masked_fill_(hidden[None, :, :, None], -math.inf)
    top = zs.amax(-1)
    zp = torch.matmul(q.reshape(G, B * n * r, D), kp).reshape(G, B, n, r, P)
    zp = _shape(zp, c, s['slopes'], P + at[:, :, None] - torch.arange(P, device=DEV) if c['slopes'] else None)
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
    row8 = D + 1                                        # a row's values and its scale
    if case['kind'] == 'read':
        return dict(bytes=2 * N * G * (row8 + 2 * D), flops=2 * N * G * D)
    if case['kind'] == 'write':
        return dict(bytes=N * (4 * D * H + 2 * G * (4 * D + row8)), flops=6 * case['pairs'] * N * (H + G) + 4 * N * G * D)
    held, window = before + new, case['window'] or 1e18
    # keys that the queries of a sequence see, and rows that at least one of them sees
    i = torch.arange(int(new.max()) + 1, dtype=torch.float64)[None, :-1]
    upto = before[:, None] + i + 1 if case['causal'] else held[:, None].expand(-1, i.shape[1])
    seen = (upto - (before[:, None] + i + 1 - window).clamp_min(0)) * (i < new[:, None])
    keys = float(seen.sum()) + N * case['prefix']
    rows = case['prefix'] + float((held - (before + 1 - window).clamp_min(0))[new > 0].sum())
    row = row8 if case['bits'] == 8 else 2 * D
    return dict(bytes=2 * D * 2 * N * H + 2 * rows * G * row + (4 * N * H if case['lse'] else 0), flops=4 * D * H * keys)


def _rounded(x):
    """float64 rows [..., 128] at the values that 8 bits hold: multiples of a step of 2^-3 of their power of two, or of
    2^-9 where that is more, times the row's own power of two."""
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** -126))))
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    lo = s['starts'].tolist()
    H, G, kind, held, table = case['heads'], case['kv_heads'], case['kind'], s['held'].tolist(), s['table'].tolist()
    if kind != 'attend':
        if case['batch'] > 400:
            return None
        got = []
        for b in range(case['batch']):
            n = lo[b + 1] - lo[b]
            rows = torch.tensor([[table[b][(held[b] + i) // PAGE], (held[b] + i) % PAGE] for i in range(n)], device=DEV,
                                dtype=torch.long).reshape(n, 2)
            if kind == 'read':
                e = s['scales'][rows[:, 0], :, :, rows[:, 1]].double() - 127
                got.append([s[x].view(torch.uint8)[rows[:, 0], :, rows[:, 1]].view(torch.float8_e4m3fn).double() *
                            (2.0 ** e[:, :, i])[..., None] for i, x in enumerate(('k8', 'v8'))])
                continue
            at = held[b] + torch.arange(n, device=DEV, dtype=torch.float64)
            pos = (at + case['first'])[:, None] if s['positions'] is None else s['positions'][lo[b]:lo[b + 1]].double()
            which = [a for a, m in enumerate(s['axes']) for _ in range(m)]
            R = len(which)
            z = torch.polar(torch.ones(n, R, dtype=torch.float64, device=DEV), pos[:, which] * s['freqs'])[:, None]

            def turned(x):
                x = x.double()
                pair = x[..., :2 * R].unflatten(-1, (R, 2) if case['interleaved'] else (2, R))
                pair = pair if case['interleaved'] else pair.transpose(-1, -2)
                w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
                w = w if case['interleaved'] else w.transpose(-1, -2)
                return torch.cat([w.flatten(-2), x[..., 2 * R:]], -1)

            part = slice(lo[b], lo[b + 1])
            dt = TYPES[case['dtype']]
            got.append([turned(s['q'][part]), _rounded(turned(s['k'][part]).to(dt).double()),
                        _rounded(s['v'][part].double())])
        return tuple(torch.cat(x) for x in zip(*got))
    if case['batch'] * G > 600:
        return None
    out = torch.zeros(s['N'], H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((s['N'], H), -math.inf, dtype=torch.float64, device=DEV)
    length, P = s['lengths'].tolist(), case['prefix']

    def rows(x, i, ids, h, count):
        ids = ids.long().clamp_min(0)
        if case['bits'] == 16:
            return s['cache_' + x][0].view(-1, PAGE, G, D)[ids, :, h].reshape(-1, D)[:count].double()
        e = s['scales'][ids, h, i].reshape(-1)[:count].double() - 127
        return s[x + '8'][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).reshape(-1, D)[:count].double() * \
            (2.0 ** e)[:, None]

    for b in range(case['batch']):
        n, own_pages = lo[b + 1] - lo[b], -(-length[b] // PAGE)
        if n == 0:
            continue
        mine = s['table'][b, :own_pages]
        at = length[b] - n + torch.arange(n, device=DEV)[:, None]
        key = torch.arange(-P, length[b], device=DEV)              # the prefix lies before row 0
        hidden = (key > at) if case['causal'] else torch.zeros(1, 1, dtype=torch.bool, device=DEV)
        if case['window']:
            hidden = hidden | (key >= 0) & (key <= at - case['window'])
        for h in range(G):
            k, v = (torch.cat([rows(x, i, s['prefix'], h, P), rows(x, i, mine, h, length[b])])
                    for i, x in enumerate('kv'))
            for hq in range(h * (H // G), (h + 1) * (H // G)):
                z = s['q'][lo[b]:lo[b + 1], hq].double() @ k.t() * D ** -0.5
                if case['cap']:
                    z = case['cap'] * torch.tanh(z / case['cap'])
                if case['slopes']:
                    z = z - s['slopes'][hq].double() * (at - key).abs()
                z = z.masked_fill(hidden, -math.inf)
                lse[lo[b]:lo[b + 1], hq] = torch.logsumexp(z, -1)
                out[lo[b]:lo[b + 1], hq] = torch.softmax(z, -1).nan_to_num(0.0) @ v
    return (out, lse) if case['lse'] else out
