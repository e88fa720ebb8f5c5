"""The 8-bit paged cache on the GPU: rows written as the 16-bit cache would hold
them and quantised, read back, and attended.

Tolerances, with u = finfo(dtype).eps / 2, half a step of the output type:
* append: a rotated element is off by less than 2^-20 (|x1| + |x2|) before its
  rounding to 16 bits (its angle by 2^-24 turns, sine, cosine and products by a few
  float32 steps); quantisation is monotone, so a value lies between those of the
  two ends, which nearly always are the same.  Rows that do not turn are exact.
* read: exact.
* attention, over the values that the cache stands for: as over 16-bit rows, the
  output's rounding u |out|, a probability's rounding at most u sum p |v| / sum p,
  a score's error below 2^-13 (128 x 2^-24 sum |q k| scale, sum |q k| scale < 16),
  float32 sums of up to n terms a lane n x 2^-24.
* lse: the scores' error and the sum's, and a step of its own.
"""
import math
import threading

import pytest
import torch

from oracle import paged as plain
from oracle import paged8 as oracle
from streaming_sparse_amd import paged, paged8
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def freqs(device, n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).to(device)


def filled(cache, seed, spread=3):
    """Random rows, their exponents within `spread` of 1's."""
    g = torch.Generator(device=cache.k.device).manual_seed(seed)
    for i, x in enumerate((cache.k, cache.v)):
        y = torch.randn(x.shape, generator=g, device=x.device)
        y = y / y.abs().amax(-1, keepdim=True) * (224 + 224 * torch.rand(y.shape[:-1], generator=g, device=x.device)[..., None])
        x.copy_(y.to(torch.float8_e4m3fn))
        # a row's largest lies at 2^8 in its own units: N(0, 1)'s at about 2^1.4
        cache.scales[:, :, i] = (120 + torch.randint(-spread if i else 0, spread + 1 if i else 1, y.shape[:-1], generator=g,
                                                     device=x.device)).to(torch.uint8)
    return cache


class Case:
    """Sequences with `new` new tokens each and `before` rows before them, pages
    anywhere in a cache whose unused rows hold NaN."""

    def __init__(self, device, new, before, heads, kv_heads, prefix=0, dtype=BF16, seed=0, padding=0, spare=2, width=None,
                 head_major=False):
        g = torch.Generator().manual_seed(seed)
        self.device, self.dtype, self.H, self.G = device, dtype, heads, kv_heads
        self.new, self.before, self.P = new, before, prefix
        self.N = sum(new)
        shared = -(-prefix // 64)
        need = [-(-(a + b) // 64) for a, b in zip(new, before)]
        width = width or max(1, max(need))
        total = shared + sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.prefix = ints(order[:shared] or [0], device)[:shared]
        rows, at = [], shared
        for n in need:
            rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.table = ints(rows, device)
        self.starts = ints([sum(new[:b]) for b in range(len(new) + 1)], device)
        self.lengths = ints([a + b for a, b in zip(new, before)], device)
        self.held = ints(before, device)
        if head_major:
            c = paged8.Cache.empty(kv_heads, total, device)
            self.cache = paged8.Cache(*(x.transpose(0, 1) for x in (c.k, c.v, c.scales)))
        else:
            self.cache = paged8.Cache.empty(total, kv_heads, device)
        filled(self.cache, seed)
        used = torch.zeros(total, 64, dtype=torch.bool)
        for pages, count in [(order[:shared], prefix)] + [(r, a + b) for r, a, b in zip(rows, new, before)]:
            for i in range(-(-count // 64)):
                used[pages[i], :min(64, count - 64 * i)] = True
        unused = ~used.to(device)
        for i, x in enumerate((self.cache.k, self.cache.v)):
            x.view(torch.uint8).masked_fill_(unused[:, None, :, None], 0x7f)         # NaN
            self.cache.scales[:, :, i].masked_fill_(unused[:, None], 255)
        self.wide = torch.randn(self.N + padding, heads + 3, 128, generator=g).to(dtype).to(device)
        self.q = self.wide[:, 1:1 + heads]

    def attend(self, causal=True, ragged=True, ws=None, **more):
        return paged8.attention(self.q, self.cache, self.prefix, self.P, self.table, self.lengths, ws or Workspace(),
                                starts=self.starts if ragged else None, causal=causal, want_lse=True, **more)

    def check(self, out, lse, causal=True, score=2.0 ** -13, **more):
        k, v = oracle.pages8(self.cache)
        want, want_lse, spread = oracle.attention(self.q, k, v, self.prefix, self.P, self.table, self.lengths, self.starts,
                                                  causal, **more)
        out, lse = out.double()[:self.N], lse.double()[:self.N]
        want, want_lse, spread = want[:self.N], want_lse[:self.N], spread[:self.N]
        u = torch.finfo(self.dtype).eps / 2
        assert torch.isfinite(out).all()
        far = (out - want).abs() - (u * want.abs() + (u + score + 2.0 ** -12) * spread + 2.0 ** -24)
        assert far.max() <= 0, float(far.max())
        none = torch.isinf(want_lse)
        assert torch.equal(none, torch.isinf(lse)) and (lse[none] < 0).all() and (out[none] == 0).all()
        off = (lse - want_lse)[~none].abs()
        assert off.numel() == 0 or (off <= score + 2.0 ** -12 + 2.0 ** -22 * want_lse[~none].abs()).all(), off.max()

    def rows(self, padding=0, seed=9):
        g = torch.Generator().manual_seed(seed)
        kv = torch.randn(self.N + padding, 2 * self.G, 128, generator=g).to(self.dtype).to(self.device)
        return kv[:, :self.G], kv[:, self.G:]


def written(c):
    """Which rows [P, 64] the new tokens take."""
    got = torch.zeros(c.cache.k.shape[0], 64, dtype=torch.bool)
    table, held, starts = c.table.tolist(), c.held.tolist(), c.starts.tolist()
    for b in range(len(held)):
        for i in range(starts[b + 1] - starts[b]):
            at = held[b] + i
            if 0 <= at < 64 * len(table[b]) and 0 <= table[b][at // 64] < got.shape[0]:
                got[table[b][at // 64], at % 64] = True
    return got.to(c.device)


def append_case(c, k, v, freqs=None, interleaved=True, first=0, axes=None, positions=None):
    before = [x.clone() for x in (c.cache.k, c.cache.v, c.cache.scales)]
    more = dict(freqs=freqs, interleaved=interleaved, first=first, axes=axes, positions=positions)
    got = paged8.append(k, v, c.cache, c.table, c.held, q=c.q, starts=c.starts, **more)
    at = torch.cat([c.held[b] + torch.arange(n, device=c.device) for b, n in enumerate(c.new)])
    b = torch.repeat_interleave(torch.arange(len(c.new), device=c.device), ints(c.new, c.device))
    page = c.table[b, (at // 64).clamp(max=c.table.shape[1] - 1)]
    there = (at < 64 * c.table.shape[1]) & (page >= 0) & (page < c.cache.k.shape[0])
    place = page[there].long(), (at % 64)[there].long()

    def both(x):
        """Rows [N, heads, 128] in 16 bits, a little less and a little more than turned."""
        if freqs is None:
            return x, x
        pos = (at + first)[:, None] if positions is None else positions
        y = plain.rotate(x.double().cpu(), pos.cpu(), freqs.cpu(), axes or (freqs.numel(),), interleaved).to(c.device)
        d = 2.0 ** -20 * x.double().abs().amax(-1, keepdim=True) * 2
        turns = (y != x.double()) | (x == 0)
        return [torch.where(turns, y + s * d * torch.sign(y), y).to(c.dtype) for s in (-1, 1)]

    low, high = (x.double() for x in both(c.q[:c.N]))
    assert ((got[:c.N].double() - low) * torch.sign(high) >= 0).all()
    assert ((high - got[:c.N].double()) * torch.sign(high) >= 0).all()
    for i, (x, new, old) in enumerate(((c.cache.k, k, before[0]), (c.cache.v, v, before[1]))):
        low, high = both(new[:c.N]) if i == 0 else (new[:c.N], new[:c.N])
        s = c.cache.scales[place[0], :, i, place[1]].long()
        assert (oracle.exponents(low)[there] <= s).all() and (s <= oracle.exponents(high)[there]).all()
        y = x.view(torch.uint8)[place[0], :, place[1]].view(torch.float8_e4m3fn).double()
        low, high = (oracle.quantise(z[there], s)[0] for z in (low, high))
        assert torch.equal(torch.isnan(y), torch.isnan(high))
        y, low, high = (z.nan_to_num() * torch.sign(high.nan_to_num()) for z in (y, low, high))
        assert ((low <= y) & (y <= high)).all()
        if freqs is None:
            assert torch.equal(low, high)
    # no other row is touched
    used = written(c)
    assert int(used.sum()) == int(there.sum())
    for i, (x, old) in enumerate(zip((c.cache.k, c.cache.v), before)):
        assert torch.equal(x.view(torch.uint8).transpose(1, 2)[~used], old.view(torch.uint8).transpose(1, 2)[~used])
        assert torch.equal(c.cache.scales[:, :, i].transpose(1, 2)[~used], before[2][:, :, i].transpose(1, 2)[~used])
    return got


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('interleaved', [True, False], ids=['pairs', 'halves'])
@pytest.mark.parametrize('pairs', [64, 40, 8])
@pytest.mark.parametrize('new,before,heads,kv_heads', [
    pytest.param([1], [0], 1, 1, id='one'),
    pytest.param([1] * 5, [0, 63, 64, 127, 1000], 8, 2, id='steps'),
    pytest.param([0, 70, 3, 0, 129], [5, 60, 0, 0, 63], 5, 3, id='ragged'),
])
def test_append(device, new, before, heads, kv_heads, pairs, interleaved, dtype):
    c = Case(device, new, before, heads, kv_heads, dtype=dtype)
    append_case(c, *c.rows(), freqs=freqs(device, pairs), interleaved=interleaved, first=1234567)


def test_append_many_tokens(device):
    c = Case(device, [3000, 1200], [10, 0], 3, 1)
    append_case(c, *c.rows(), freqs=freqs(device, 64))


def test_append_axes(device):
    c = Case(device, [40, 25], [0, 7], 4, 4)
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (c.N, 3), generator=torch.Generator().manual_seed(4)).to(torch.int32).to(device)
    f = torch.cat([freqs(device, n) for n in (22, 21, 21)])
    append_case(c, *c.rows(), freqs=f, axes=(22, 21, 21), positions=pos)


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
def test_append_every_value(device, dtype):
    """Every 16-bit value, in rows whose largest is anything: the ends of the type,
    subnormals, zeros of either sign, infinities and NaN among them."""
    every = torch.arange(-32768, 32768).to(torch.int16).view(dtype)
    g = torch.Generator().manual_seed(1)
    order = torch.cat([torch.arange(65536), torch.randperm(65536, generator=g), every.double().nan_to_num(0, 0, 0).abs().argsort()])
    rows = every[order].reshape(-1, 2, 128)
    finite = torch.where(torch.isfinite(rows.double()), rows.double(), 0.0).to(dtype)      # rows without a NaN, too
    rows = torch.cat([rows, finite, torch.zeros(2, 2, 128, dtype=dtype)]).to(device)
    c = Case(device, [len(rows)], [0], 1, 2, dtype=dtype)
    append_case(c, rows, rows.flip(0))


def test_append_borders_of_the_power_of_two(device):
    """A row's largest at, below and above 448 times a power of two, and values half
    way between two of those held."""
    for dtype in (BF16, FP16):
        x = torch.zeros(24, 1, 128)
        for i in range(24):
            top = 448.0 * 2.0 ** (i % 8 - 6)
            step = top * torch.finfo(dtype).eps
            x[i, 0, i] = (top - step, top, top + step)[i // 8] * (-1) ** i
            x[i, 0, 64:] = torch.arange(64) * top / 448 * 2.0 ** -4
        c = Case(device, [24], [0], 1, 1, dtype=dtype)
        x = x.to(dtype).to(device)
        append_case(c, x, -x)


def test_append_outside_the_table_or_cache(device):
    c = Case(device, [4, 70], [60, 0], 2, 1, padding=5)
    c.table[1, 1] = -1
    c.held = ints([126, 0], device)
    k, v = c.rows(padding=5)
    q_out = torch.full_like(c.q, 3.0)
    append_case(c, k, v)
    got = paged8.append(k, v, c.cache, c.table, c.held, q=c.q, q_out=q_out, starts=c.starts)
    assert got is q_out and (got[c.N:] == 3.0).all() and torch.equal(got[:c.N], c.q[:c.N])


def test_append_head_major_and_sliced(device):
    """Pages in another order in memory, and a slice of a larger cache's heads."""
    c = Case(device, [7, 80], [60, 3], 3, 2, head_major=True)
    append_case(c, *c.rows(), freqs=freqs(device, 48), interleaved=False)
    big = filled(paged8.Cache.empty(9, 5, device), 1)
    c = Case(device, [7, 80], [60, 3], 3, 2)
    assert c.cache.k.shape[0] <= 9
    c.cache = paged8.Cache(big.k[:, 1:3], big.v[:, 1:3], big.scales[:, 1:3])
    append_case(c, *c.rows())


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('new,first,kv_heads', [
    pytest.param([1], [0], 1, id='one'),
    pytest.param([1] * 5, [0, 63, 64, 127, 1000], 2, id='steps'),
    pytest.param([0, 70, 3, 0, 129], [5, 60, 0, 0, 63], 3, id='ragged'),
    pytest.param([2500], [77], 12, id='long'),
    pytest.param([0 if i % 5 < 2 else 1 + i % 2 for i in range(300)], [(7 * i) % 100 for i in range(300)], 1, id='many'),
])
def test_read(device, new, first, kv_heads, dtype):
    """The values that the cache stands for, rounded once to fp16, unrounded in bf16."""
    c = Case(device, new, first, 1, kv_heads)
    k, v = paged8.read(c.cache, c.table, c.held, c.N, starts=c.starts, dtype=dtype)
    new_rows = written(c)
    for got, want in zip((k, v), oracle.pages8(c.cache)):
        assert got.dtype is dtype and got.shape == (c.N, kv_heads, 128)
        table, starts = c.table.tolist(), c.starts.tolist()
        place = [(table[b][(first[b] + i) // 64], (first[b] + i) % 64) for b in range(len(new)) for i in range(new[b])]
        page, row = torch.tensor(place, device=device).reshape(-1, 2).t()
        rows = want[page, :, row]
        assert torch.equal(got, rows.to(dtype))
        if dtype is BF16:
            assert torch.equal(got.double(), rows)
    assert int(new_rows.sum()) == c.N


def test_read_absent_rows_and_padding(device):
    """Zeros for rows outside the table or the cache, nothing behind the last sequence;
    into rows of a 16-bit cache."""
    c = Case(device, [8, 70], [120, 0], 1, 2)
    c.table[1, 1] = -1
    # two more rows of the first sequence, behind its table
    c.new, c.N, c.starts = [10, 70], 80, ints([0, 10, 80], device)
    total = c.N + 7
    k_out = torch.full((total, 5, 128), 9.0, dtype=BF16, device=device)
    v_out = torch.full((2, total, 128), 9.0, dtype=BF16, device=device).transpose(0, 1)
    k, v = paged8.read(c.cache, c.table, c.held, total, starts=c.starts, k_out=k_out[:, 1:3], v_out=v_out)
    for x in (k, v):
        assert (x[c.N:] == 9.0).all() and (x[8:10] == 0).all() and (x[10 + 64:c.N] == 0).all()
        assert (x[:8].float().abs().sum(-1) > 0).all() and (x[10:74].float().abs().sum(-1) > 0).all()
    assert (k_out[:, 0] == 9.0).all() and (k_out[:, 3:] == 9.0).all()
    resident = torch.full((1, 64 * 4, 2, 128), 9.0, dtype=BF16, device=device)
    other = resident.clone()
    got, _ = paged8.read(c.cache, c.table[:1], c.held[:1], 8, k_out=resident[0, 64:72], v_out=other[0, 64:72])
    assert torch.equal(got, k[:8]) and (resident[0, :64] == 9.0).all() and (resident[0, 72:] == 9.0).all()


SHAPES = [
    # new tokens, rows before them, heads, K/V heads, prefix
    pytest.param([1], [0], 1, 1, 0, id='one_key'),
    pytest.param([1], [0], 2, 1, 1, id='two_keys'),
    pytest.param([1], [62], 3, 3, 0, id='page_full'),
    pytest.param([1, 1, 1], [63, 64, 31], 4, 4, 130, id='steps_shared'),
    pytest.param([1] * 9, list(range(0, 270, 30)), 8, 2, 1003, id='steps_gqa'),
    pytest.param([1] * 70, [3 * i for i in range(70)], 7, 1, 321, id='steps_mqa_70'),
    pytest.param([1], [4000], 4, 1, 1500, id='step_long'),
    pytest.param([5, 5, 5, 5], [7, 0, 300, 64], 4, 2, 700, id='verify'),
    pytest.param([0, 3, 1, 0, 17], [5, 61, 0, 0, 128], 6, 3, 65, id='ragged_zero'),
    pytest.param([33, 100, 2], [0, 31, 129], 4, 1, 64, id='ragged_gqa'),
    pytest.param([130], [70], 3, 3, 190, id='prompt'),
    pytest.param([129, 64], [0, 1], 2, 2, 0, id='no_prefix'),
    pytest.param([257], [0], 5, 1, 449, id='prompt_mqa'),
    pytest.param([300, 1, 200], [10, 900, 0], 2, 2, 515, id='mixed'),
]


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('causal', [True, False], ids=['causal', 'full'])
@pytest.mark.parametrize('new,before,heads,kv_heads,prefix', SHAPES)
def test_attention(device, new, before, heads, kv_heads, prefix, causal, dtype):
    c = Case(device, new, before, heads, kv_heads, prefix, dtype)
    c.check(*c.attend(causal), causal)


@pytest.mark.parametrize('batch,new,held,heads,kv_heads,prefix,causal,dtype', [
    # every way through the kernels
    pytest.param(8, 1, 200, 8, 8, 9000, True, BF16, id='apart_narrow'),
    pytest.param(11, 1, 200, 12, 4, 9000, True, BF16, id='apart_two_narrow_33'),
    pytest.param(21, 1, 700, 6, 2, 20000, False, FP16, id='apart_two_narrow_63'),
    pytest.param(9, 1, 200, 3, 1, 5000, True, FP16, id='joint_narrow_pieces'),
    pytest.param(1, 1, 30, 8, 2, 30000, True, BF16, id='joint_narrow_many_pieces'),
    pytest.param(40, 3, 400, 12, 12, 0, True, FP16, id='joint_narrow_whole'),
    pytest.param(90, 1, 700, 6, 2, 20000, True, BF16, id='apart_wide_many_pieces'),
    pytest.param(30, 7, 90, 14, 2, 700, True, FP16, id='wide_few_tokens'),
    pytest.param(300, 1, 130, 16, 8, 700, True, BF16, id='apart_items_in_turn'),
    pytest.param(1, 200, 50, 8, 2, 30000, True, BF16, id='joint_wide_many_pieces'),
    pytest.param(3, 601, 7, 8, 8, 126, True, FP16, id='half_wide_whole'),
    pytest.param(1, 1265, 134, 12, 4, 248, True, BF16, id='half_wide_causal_cut'),
    pytest.param(2, 700, 0, 48, 48, 1000, False, BF16, id='joint_wide_rounds'),
    pytest.param(1, 2000, 100, 12, 12, 10, True, BF16, id='causal_cut'),
    pytest.param(5, 530, 1600, 8, 1, 4300, False, BF16, id='prompts'),
])
def test_attention_large(device, batch, new, held, heads, kv_heads, prefix, causal, dtype):
    before = torch.randint(0, held + 1, (batch,), generator=torch.Generator().manual_seed(4)).tolist()
    c = Case(device, [new] * batch, before, heads, kv_heads, prefix, dtype)
    ws = Workspace()
    out, lse = (x.clone() for x in c.attend(causal, ragged=False, ws=ws))
    # a lane adds up to 16384 of its row's probabilities one by one: 2^-10 relative, 2^-12 of it allowed anyway
    c.check(out, lse, causal, score=2.0 ** -13 + 2.0 ** -10)
    again = c.attend(causal, ragged=False, ws=ws)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for parts in (True, False):
        c.check(*c.attend(causal, single_av=parts), causal, score=2.0 ** -13 + 2.0 ** -10)


@pytest.mark.parametrize('new,held,heads,kv_heads,prefix', [
    pytest.param([1] * 70, 100, 8, 2, 2500, id='apart'),
    pytest.param([150, 90], 70, 3, 1, 321, id='joint'),
    pytest.param([1] * 6, 300, 4, 2, 2500, id='narrow_apart'),
    pytest.param([1], 3000, 4, 2, 0, id='narrow'),
    pytest.param([2] * 3, 500, 8, 2, 321, id='narrow_joint'),
])
@pytest.mark.parametrize('powers', ['alike', 'rising', 'falling', 'one_page', 'one_row', 'one_row_near', 'first_page', 'wide_apart', 'tiny',
                                    'huge', 'zeros', 'edges'])
def test_attention_powers_of_two_of_values(device, new, held, heads, kv_heads, prefix, powers):
    """Tiles with two parts hold the values relative to the largest power of two so far
    where that is exact: rows within and outside that range, in any order."""
    c = Case(device, new, [held] * len(new), heads, kv_heads, prefix)
    s = c.cache.scales[:, :, 1]
    live = s != 255
    order = c.prefix.tolist()
    at = torch.zeros(s.shape[0], dtype=torch.long, device=device)           # a page's place in its list
    for i, p in enumerate(order):
        at[p] = i
    for row in c.table.tolist():
        for i, p in enumerate(row):
            if p >= 0:
                at[p] = len(order) + i
    place = 64 * at[:, None] + torch.arange(64, device=device)              # [P, 64]
    e = torch.full_like(place, 124)
    if powers == 'rising':
        e = 60 + place // 24
    elif powers == 'falling':
        e = 200 - place // 24
    elif powers == 'one_page':
        e = torch.where(at[:, None] == 3, 100 + torch.arange(64, device=device), e)
    elif powers == 'one_row':                   # one that no query gives weight
        e = torch.where(place == 200, 240, e)
    elif powers == 'one_row_near':              # and the others just within its range: fp16's smallest values
        e = torch.where(place == 200, 139, e)
    elif powers == 'first_page':
        e = torch.where(at[:, None] == 0, torch.arange(64, device=device) * 3 + 40, e)
    elif powers == 'wide_apart':
        e = torch.where(place % 2 == 0, 30, 230)
    elif powers == 'tiny':
        e = torch.full_like(place, 3) + place % 9
    elif powers == 'huge':
        e = torch.full_like(place, 225) + place % 9
    elif powers == 'edges':                     # just inside the range of one power and just outside it
        e = torch.where(at[:, None] < 3, 124 - place % 16, 124 - place % 17)
    s.copy_(torch.where(live, e.to(torch.uint8)[:, None].expand_as(s), s))
    if powers == 'zeros':
        zero = live & (place % 5 == 0)[:, None]
        c.cache.v.view(torch.uint8).masked_fill_(zero[..., None], 0)
        s.masked_fill_(zero, 1)
    if powers.startswith('one_row'):
        page = (order + c.table[0].tolist())[200 // 64]
        # every query's score with it is about -317, others' within 16 of 0
        c.q[:] = 4.0 * (0.25 + 0.01 * c.q)
        c.cache.k[page, :, 200 % 64] = -448.0
        c.cache.scales[page, :, 0, 200 % 64] = 123
    for single in (False, None):
        c.check(*c.attend(single_av=single), score=2.0 ** -13 + 2.0 ** -10)


def test_attention_powers_of_two_far_apart(device):
    """Values from 2^-80 to 2^80 in rows next to each other, keys whose powers
    nearly cancel the queries': the largest rule, nothing is lost or infinite."""
    for new in ([1, 1], [150]):
        c = Case(device, new, [200] * len(new), 2, 2, 300)
        live = c.cache.scales != 255
        g = torch.Generator(device=device).manual_seed(5)
        s = torch.randint(40, 200, c.cache.scales[:, :, 1].shape, generator=g, device=device).to(torch.uint8)
        c.cache.scales[:, :, 1] = torch.where(live[:, :, 1], s, c.cache.scales[:, :, 1])
        # keys times 2^-100, the scale 2^100 of what it was
        c.cache.scales[:, :, 0] -= 100 * live[:, :, 0].to(torch.uint8)
        out, lse = c.attend(scale=128 ** -0.5 * 2.0 ** 100)
        c.check(out, lse, scale=128 ** -0.5 * 2.0 ** 100)


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
def test_attention_is_that_over_the_rows_read(device, dtype):
    """The 16-bit attention over the rows that `read` returns gives the same, up to
    both sides' roundings."""
    for new, before in (([1] * 6, [300] * 6), ([90, 40], [20, 130])):
        c = Case(device, new, before, 4, 2, 0, dtype)
        k, v = (c.cache.k, c.cache.v)
        got, lse = c.attend()
        counts = c.lengths.tolist()
        starts = ints([sum(counts[:b]) for b in range(len(counts) + 1)], device)
        rk, rv = paged8.read(c.cache, c.table, torch.zeros_like(c.held), sum(counts), starts=starts, dtype=dtype)
        ck, cv = (torch.zeros(1, 64 * k.shape[0], 2, 128, dtype=dtype, device=device) for _ in range(2))
        paged.append(rk, rv, ck, cv, c.table, torch.zeros_like(c.held), starts=starts)
        want, want_lse = paged.attention(c.q, ck, cv, None, 0, c.table, c.lengths, Workspace(), starts=c.starts,
                                         want_lse=True)
        u = torch.finfo(dtype).eps / 2
        size = cv.abs().max().double()
        assert ((got.double() - want.double()).abs() <= 2 * u * want.double().abs() + (2 * u + 2.0 ** -11) * size).all()
        assert ((lse - want_lse).abs() <= 2.0 ** -12).all()


def test_attention_leaves_rows_behind_the_last_sequence(device):
    c = Case(device, [4, 9], [0, 70], 3, 1, 90, padding=6)
    out = torch.full_like(c.q, 7.0)
    got, lse = c.attend(out=out)
    c.check(got, lse)
    assert got is out and (out[c.N:] == 7.0).all()


def test_attention_rows_that_see_nothing(device):
    for new in ([6, 2], [200, 3]):
        c = Case(device, new, [0, 0], 2, 1, 0)
        c.lengths = ints([4, 0], device)
        out, lse = c.attend()
        c.check(out, lse)
        assert (out[:new[0] - 4] == 0).all() and torch.isinf(lse[:new[0] - 4]).all()


def test_attention_absent_pages(device):
    for new in ([2, 2], [200, 90]):
        c = Case(device, new, [300, 200], 2, 2, 330)
        c.prefix[1] = -1
        c.prefix[5] = 1 << 20
        c.table[0, 0] = -7
        c.table[1, 3] = -1
        c.check(*c.attend())
        c.prefix[:] = -1
        c.table[1, :] = -1
        c.check(*c.attend())


@pytest.mark.parametrize('causal', [True, False], ids=['causal', 'full'])
@pytest.mark.parametrize('new,before,heads,kv_heads,prefix,drop', [
    pytest.param([4], [126], 2, 2, 0, 1, id='narrow'),
    pytest.param([1] * 40, [64 + 7 * i for i in range(40)], 2, 1, 300, 3, id='wide_shared'),
    pytest.param([300, 40], [10, 250], 2, 2, 70, 2, id='wide'),
])
def test_attention_lengths_past_the_table(device, new, before, heads, kv_heads, prefix, drop, causal):
    c = Case(device, new, before, heads, kv_heads, prefix)
    c.table = c.table[:, :max(1, c.table.shape[1] - drop)].contiguous()
    assert int(c.lengths.max()) > 64 * c.table.shape[1]
    c.check(*c.attend(causal), causal)


def test_attention_layouts(device):
    """Head-major pages, a slice of a larger cache's heads, head-major and broadcast
    queries, out in place of q, garbage behind the table's used entries."""
    c = Case(device, [5, 40], [100, 3], 4, 2, 200, width=9)
    want, want_lse = (x.clone() for x in c.attend())
    pages = c.cache.k.shape[0]
    flipped = paged8.Cache(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (c.cache.k, c.cache.v, c.cache.scales)))
    big = paged8.Cache.empty(pages, 5, device)
    sliced = paged8.Cache(big.k[:, 2:4], big.v[:, 2:4], big.scales[:, 2:4])
    for a, b in zip((sliced.k, sliced.v, sliced.scales), (c.cache.k, c.cache.v, c.cache.scales)):
        a.view(torch.uint8).copy_(b.view(torch.uint8))
    used = -(-c.lengths // 64)
    c.table[torch.arange(9, device=device) >= used[:, None]] = 0x7fffffff
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    for cache in (flipped, sliced):
        c.cache = cache
        got, lse = c.attend()
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
    got, lse = c.attend(out=c.q)
    assert got is c.q and torch.equal(got, want) and torch.equal(lse, want_lse)


def test_attention_nan_reaches_only_who_sees_it(device):
    c = Case(device, [1, 1], [100, 100], 2, 1, 100)
    pg = int(c.table[0, 0])
    c.cache.k.view(torch.uint8)[pg, 0, 5, 3] = 0x7f
    out, _ = c.attend()
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_attention_masked_nan_key(device):
    for new, before in (([7], [60]), ([300], [5])):
        c = Case(device, new, before, 2, 2, 70)
        want = c.attend()[0].clone()
        for at in (c.lengths[0] - 1, c.lengths[0] - 2):
            c.cache.k.view(torch.uint8)[int(c.table[0, int(at) // 64]), :, int(at) % 64, 0] = 0x7f
        got, _ = c.attend()
        assert torch.equal(got[:c.N - 2], want[:c.N - 2]) and torch.isnan(got[c.N - 2:]).all()


def test_cache_offsets_past_32_bits(device):
    """Pages beyond 2^32 bytes of a cache."""
    G, pages = 64, 8400                      # 64 x 8192 bytes a page: 4.4e9
    k, v = (torch.zeros(pages, G, 64, 128, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
    cache = paged8.Cache(k, v, torch.full((pages, G, 2, 64), 120, dtype=torch.uint8, device=device))
    table = ints([[pages - 1, 1], [pages - 2, pages - 3]], device)
    held, lengths = ints([3, 64], device), ints([5, 66], device)
    few = [pages - 1, pages - 2, pages - 3, pages - 4]
    part = filled(paged8.Cache.empty(4, G, device), 1)
    for i, pg in enumerate(few):
        k.view(torch.uint8)[pg], v.view(torch.uint8)[pg] = part.k[i].view(torch.uint8), part.v[i].view(torch.uint8)
        cache.scales[pg] = part.scales[i]
    rows = torch.randn(4, 3 * G, 128, generator=torch.Generator(device=device).manual_seed(1), device=device).to(BF16)
    q, kk, vv = rows[:, :G], rows[:, G:2 * G], rows[:, 2 * G:]
    paged8.append(kk, vv, cache, table, held)
    got_k, got_v = paged8.read(cache, table, held, 4)
    for got, x in ((got_k, kk), (got_v, vv)):
        want, s = oracle.quantise(x)
        assert torch.equal(got.double(), oracle.values(want, s))
    prefix = ints([pages - 4], device)
    out = paged8.attention(q, cache, prefix, 50, table, lengths, Workspace())
    small = paged8.Cache(*(torch.stack([x[p] for p in few + [1]]) for x in (k.view(torch.uint8), v.view(torch.uint8),
                                                                            cache.scales)))
    small.k, small.v = (x.view(torch.float8_e4m3fn) for x in (small.k, small.v))
    want, _, spread = oracle.attention(q, *oracle.pages8(small), ints([3], device), 50, ints([[0, 4], [1, 2]], device),
                                       lengths, torch.tensor([0, 2, 4]))
    u = torch.finfo(BF16).eps / 2
    assert ((out.double() - want).abs() <= u * want.abs() + (u + 2.0 ** -11) * spread + 2.0 ** -24).all()


def test_steps_of_several_sequences(device):
    """As they are used: a common prompt, three sequences that append and attend
    token by token, their rows handed back; equal to the whole of each at once."""
    H, G, P, B, steps = 4, 2, 150, 3, 70
    c = Case(device, [0] * B, [0] * B, H, G, P, width=2, spare=2 * B)
    free = [p for p in range(c.cache.k.shape[0]) if p not in c.prefix.tolist()]
    c.table = ints([free[2 * b:2 * b + 2] for b in range(B)], device)
    rows = torch.randn(steps, B, H + 2 * G, 128, generator=torch.Generator().manual_seed(2)).to(BF16).to(device)
    f, ws = freqs(device, 64), Workspace()
    held = ints([0] * B, device)
    outs = []
    for s in range(steps):
        q, k, v = rows[s, :, :H], rows[s, :, H:H + G], rows[s, :, H + G:]
        q = paged8.append(k, v, c.cache, c.table, held, q=q, freqs=f, first=P, workspace=ws)
        held += 1
        outs.append(paged8.attention(q, c.cache, c.prefix, P, c.table, held, ws).clone())
    got = torch.stack(outs, 1).reshape(B * steps, H, 128)
    zero = ints([0] * B, device)
    step_k, step_v = paged8.read(c.cache, c.table, zero, B * steps)
    # the same at once, in an empty copy of the cache
    other = paged8.Cache(*(x.view(torch.uint8).clone() for x in (c.cache.k, c.cache.v, c.cache.scales)))
    for pg in c.table.flatten().tolist():
        other.k[pg], other.v[pg], other.scales[pg] = 0x7f, 0x7f, 255
    other.k, other.v = other.k.view(torch.float8_e4m3fn), other.v.view(torch.float8_e4m3fn)
    flat = rows.transpose(0, 1).reshape(B * steps, H + 2 * G, 128)
    q = paged8.append(flat[:, H:H + G], flat[:, H + G:], other, c.table, zero, q=flat[:, :H], freqs=f, first=P)
    all_k, all_v = paged8.read(other, c.table, zero, B * steps)
    assert torch.equal(step_k, all_k) and torch.equal(step_v, all_v)
    out = paged8.attention(q, other, c.prefix, P, c.table, held, Workspace())
    want, _, spread = oracle.attention(q, *oracle.pages8(other), c.prefix, P, c.table, held, torch.arange(B + 1) * steps)
    u = torch.finfo(BF16).eps / 2
    for x in (got, out):
        assert ((x.double() - want).abs() <= u * want.abs() + (u + 2.0 ** -11) * spread + 2.0 ** -24).all()


def test_captured_step_replays_with_new_lengths(device):
    """Append, read back and attention captured in a graph and replayed token by token,
    eager work between: every replay equals the eager calls bit for bit."""
    c = Case(device, [1] * 6, [0, 5, 63, 64, 100, 126], 8, 2, 700, width=3)
    total = c.cache.k.shape[0]
    cache = filled(paged8.Cache.empty(total + 18, 2, device), 3)
    table = (total + torch.arange(18, device=device, dtype=torch.int32)).reshape(6, 3)
    rows = torch.empty(6, 12, 128, dtype=BF16, device=device)
    held, lengths = c.held.clone(), c.held + 1
    f = freqs(device, 64)

    def step(ws, cache):
        q = paged8.append(rows[:, 8:10], rows[:, 10:], cache, table, held, q=rows[:, :8], freqs=f, first=700, workspace=ws)
        k, v = paged8.read(cache, table, held, 6, workspace=ws)
        return (*paged8.attention(q, cache, c.prefix, 700, table, lengths, ws, want_lse=True), k, v)

    def fill(s):
        rows.copy_(torch.randn(6, 12, 128, generator=torch.Generator().manual_seed(s)).to(BF16))

    fill(0)
    ws, eager_ws = Workspace(), Workspace()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ws, cache)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(ws, cache)
    eager = paged8.Cache(*(x.view(torch.uint8).clone() for x in (cache.k, cache.v, cache.scales)))
    eager.k, eager.v = eager.k.view(torch.float8_e4m3fn), eager.v.view(torch.float8_e4m3fn)
    for s in range(1, 5):
        fill(s)
        held += 13
        lengths.copy_(held + 1)
        torch.randn(1 << 20, device=device).sum()
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager_ws, eager)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for x in ('k', 'v', 'scales'):
            assert torch.equal(getattr(cache, x).view(torch.uint8), getattr(eager, x).view(torch.uint8))


def test_in_place_and_two_threads(device):
    """Two threads that call with different sizes at once, each on a stream and with a
    workspace of its own, over 8-bit and 16-bit caches in turn."""
    cs = [Case(device, [1] * 12, [50 * i for i in range(12)], 8, 2, 3000, seed=1),
          Case(device, [300, 1, 200], [10, 900, 0], 2, 2, 515, seed=2), Case(device, [1], [200], 4, 4, 0, seed=3),
          Case(device, [700], [30], 8, 1, 0, seed=4)]
    want = [tuple(x.clone() for x in c.attend()) for c in cs]
    torch.cuda.synchronize()
    failed = []

    def calls(order):
        try:
            ws, stream = Workspace(), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in order * 5:
                    out, lse = cs[i].attend(ws=ws)
                    stream.synchronize()
                    if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])):
                        failed.append(i)
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=calls, args=(o,)) for o in ([0, 1, 2, 3], [3, 1, 0, 2])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_no_rows_at_all(device):
    for new in ([0, 0, 0], [0]):
        c = Case(device, new, [70] * len(new), 2, 1, 90, padding=9)
        out = torch.full_like(c.q, 5.0)
        got, _ = c.attend(out=out)
        assert (got == 5.0).all()
        k = torch.full((9, 1, 128), 5.0, dtype=BF16, device=device)
        paged8.read(c.cache, c.table, c.held, 9, starts=c.starts, k_out=k, v_out=k.clone())
        assert (k == 5.0).all()


def test_values_that_the_cache_stands_for_stay_within_their_error(device):
    """A value is off by at most 2^-4 of itself, or 2^-17 of the row's largest (half a
    step of 2^-9 beside a largest of more than 224)."""
    c = Case(device, [500], [0], 1, 3)
    k, v = c.rows()
    k = k * torch.exp2(6 * torch.randn(k.shape, generator=torch.Generator(device=device).manual_seed(2), device=device))
    paged8.append(k.to(BF16), v, c.cache, c.table, c.held)
    got, _ = paged8.read(c.cache, c.table, c.held, 500)
    x = k.to(BF16).double()
    assert ((got.double() - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), x.abs().amax(-1, keepdim=True) * 2.0 ** -17)).all()
    assert math.isfinite(float(got.double().norm()))
