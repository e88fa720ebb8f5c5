"""Paged append and shared-prefix attention on the GPU against the float64
oracle.

Tolerances, with u = finfo(dtype).eps / 2, half a step of the output type:
* append: a result is rounded once (u |y|); its angle is off by at most
  2^-24 turns and the sine, cosine and products by a few float32 steps, all
  below 2^-20 (|x1| + |x2|).
* attention: the output's rounding (u |out|); a probability's rounding to 16
  bits is relative, so it moves the output by at most u sum p |v| / sum p; a
  score is a float32 sum of 128 products and is off by less than 128 x 2^-24
  sum |q k| scale < 2^-13 at these inputs (sum |q k| scale < 16), and so is,
  relatively, a probability; the float32 sums over at most 6000 keys add
  less than 3000 x 2^-24 < 2^-12 in the worst order.
* lse: the scores' error and the sum's, 2^-13 + 2^-12, and a step of its own.
"""
import math
import threading

import pytest
import torch

from oracle import paged as oracle
from streaming_sparse_amd import _lib, paged
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Case:
    """Sequences with `new` new tokens each and `before` rows before them, pages
    anywhere in a cache whose unused rows hold NaN."""

    def __init__(self, device, new, before, heads, kv_heads, prefix=0, dtype=BF16, seed=0, padding=0, head_major=False,
                 spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.device, self.dtype, self.H, self.G = device, dtype, heads, kv_heads
        self.new, self.before, self.P = new, before, prefix
        B = len(new)
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
        self.starts = ints([sum(new[:b]) for b in range(B + 1)], device)
        self.lengths = ints([a + b for a, b in zip(new, before)], device)
        self.held = ints(before, device)
        shape = (kv_heads, 64 * total, 128) if head_major else (64 * total, kv_heads, 128)

        def cache():
            x = torch.full(shape, math.nan, dtype=dtype, device=device)
            return (x.transpose(0, 1) if head_major else x)[None]

        self.k, self.v = cache(), cache()
        for pages, count in [(order[:shared], prefix)] + [(r, a + b) for r, a, b in zip(rows, new, before)]:
            for i in range(-(-count // 64)):
                m = min(64, count - 64 * i)
                for x in (self.k, self.v):
                    x[0, 64 * pages[i]:64 * pages[i] + m] = torch.randn(m, kv_heads, 128, generator=g).to(dtype).to(device)
        # queries as a part of a wider projection
        self.wide = torch.randn(self.N + padding, heads + 3, 128, generator=g).to(dtype).to(device)
        self.q = self.wide[:, 1:1 + heads]

    def attend(self, causal=True, ragged=True, want_lse=True, ws=None, **more):
        return paged.attention(self.q, self.k, self.v, self.prefix, self.P, self.table, self.lengths,
                               ws or Workspace(), starts=self.starts if ragged else None, causal=causal,
                               want_lse=want_lse, **more)

    def check(self, out, lse, causal=True, scale=None):
        want, want_lse, spread = oracle.attention(self.q, self.k, self.v, self.prefix, self.P, self.table,
                                                  self.lengths, self.starts, causal, scale)
        out, lse = out.cpu().double()[:self.N], lse.cpu().double()[:self.N]
        want, want_lse, spread = want[:self.N], want_lse[:self.N], spread[:self.N]
        u = torch.finfo(self.dtype).eps / 2
        assert torch.isfinite(out).all()
        far = (out - want).abs() - (u * want.abs() + (u + 2.0 ** -13 + 2.0 ** -12) * spread + 2.0 ** -24)
        assert far.max() <= 0, float(far.max())
        none = torch.isinf(want_lse)
        assert torch.equal(none, torch.isinf(lse)) and (lse[none] < 0).all() and (out[none] == 0).all()
        off = (lse - want_lse)[~none].abs()
        assert off.numel() == 0 or (off <= 2.0 ** -13 + 2.0 ** -12 + 2.0 ** -22 * want_lse[~none].abs()).all(), off.max()


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


def test_attention_equal_counts_need_no_starts(device):
    c = Case(device, [3, 3, 3], [10, 64, 200], 4, 2, 130)
    a, b = c.attend(ragged=True), c.attend(ragged=False)
    c.check(*b)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_head_major_cache_and_scale(device):
    c = Case(device, [2, 90], [100, 5], 4, 2, 200, head_major=True)
    c.check(*c.attend(scale=0.05), scale=0.05)


def test_attention_leaves_rows_behind_the_last_sequence(device):
    c = Case(device, [4, 9], [0, 70], 3, 1, 90, padding=6)
    out = torch.full_like(c.q, 7.0)
    got, lse = c.attend(out=out)
    c.check(got, lse)
    assert got is out and (out[c.N:] == 7.0).all()


def test_attention_rows_that_see_nothing(device):
    """No prefix and fewer rows in the cache than new tokens: with `causal` the
    first ones see none; an empty sequence sees none at all."""
    c = Case(device, [6, 2], [0, 0], 2, 1, 0)
    c.lengths = ints([4, 0], device)
    out, lse = c.attend()
    c.check(out, lse)
    assert (out[:2] == 0).all() and torch.isinf(lse[:2]).all() and torch.isfinite(lse[2:6]).all()


def test_attention_absent_pages(device):
    """Pages outside the cache count as absent, in the prefix, in a table, first
    and last."""
    c = Case(device, [2, 2], [300, 200], 2, 2, 330)
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
    pytest.param([1, 5, 2], [70, 190, 3], 4, 2, 130, 2, id='narrow_shared'),
    pytest.param([1] * 40, [64 + 7 * i for i in range(40)], 2, 1, 300, 3, id='wide_shared'),
    pytest.param([300, 40], [10, 250], 2, 2, 70, 2, id='wide'),
    pytest.param([257], [3], 1, 1, 0, 4, id='wide_few_rows_left'),
])
def test_attention_lengths_past_the_table(device, new, before, heads, kv_heads, prefix, drop, causal):
    """Tokens that were not written, their rows outside the table: the others keep
    the rows that they see, whatever the length is."""
    c = Case(device, new, before, heads, kv_heads, prefix)
    c.table = c.table[:, :max(1, c.table.shape[1] - drop)].contiguous()
    assert int(c.lengths.max()) > 64 * c.table.shape[1]
    c.check(*c.attend(causal), causal)
    # no query misses a row that it should see, up to the largest length there is
    # (the longest sequence's, whose rows fill the table)
    c.lengths[c.lengths.argmax()] = 2 ** 31 - 1
    c.check(*c.attend(causal), causal)


def test_attention_wide_table_and_repeated_pages(device):
    """A table wider than any sequence, and sequences that share own pages."""
    c = Case(device, [1, 1, 1], [100, 140, 20], 4, 4, 64, width=40)
    c.table[1, 0] = c.table[0, 0]
    c.check(*c.attend())


def test_attention_large_scores(device):
    """Scores far apart: one key holds all the weight; maxima grow along the list
    (the accumulator is rescaled) or fall."""
    for sign in (1.0, -1.0):
        c = Case(device, [3], [900], 2, 2, 900, dtype=FP16)
        ramp = torch.linspace(-1, 1, 64 * (c.k.shape[1] // 64), device=device) * 3 * sign
        for pages in (c.prefix.tolist(), c.table[0].tolist()):
            for i, pg in enumerate(pages):
                c.k[0, 64 * pg:64 * pg + 64, :, :64] = ((i * 64 + torch.arange(64, device=device)) / 300 * sign)[:, None, None]
        c.q[..., :64] = 1.0
        out, lse = c.attend()
        want, want_lse, spread = oracle.attention(c.q, c.k, c.v, c.prefix, c.P, c.table, c.lengths, c.starts)
        # a score of up to 90 is a float32 sum of 128 products: 128 x 2^-24 x 90 < 2^-10
        u = torch.finfo(FP16).eps / 2
        assert ((out.cpu().double() - want).abs() <= u * want.abs() + (u + 2.0 ** -10 + 2.0 ** -12) * spread + 2.0 ** -24).all()
        assert ((lse.cpu().double() - want_lse).abs() <= 2.0 ** -10 + 2.0 ** -12).all()


def test_attention_nan_and_inf_reach_only_who_sees_them(device):
    """A NaN key of one sequence's own rows makes that sequence's rows NaN and no
    other's."""
    c = Case(device, [1, 1], [100, 100], 2, 1, 100)
    pg = int(c.table[0, 0])
    c.k[0, 64 * pg + 5] = math.nan
    out, _ = c.attend()
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_attention_masked_nan_key(device):
    """Keys of later tokens are masked whatever they hold: with NaN keys in the
    last two tokens the earlier rows stay as they are."""
    for new, before in (([7], [60]), ([300], [5])):
        c = Case(device, new, before, 2, 2, 70)
        want, _ = c.attend()
        want = want.clone()
        for at in (c.lengths[0] - 1, c.lengths[0] - 2):
            c.k[0, 64 * int(c.table[0, int(at) // 64]) + int(at) % 64] = math.nan
        got, _ = c.attend()
        assert torch.equal(got[:c.N - 2], want[:c.N - 2]) and torch.isnan(got[c.N - 2:]).all()


@pytest.mark.parametrize('new,before,heads,kv_heads,prefix', [
    pytest.param([1], [3], 2, 2, 1300, id='narrow_pieces'),
    pytest.param([1, 1, 2], [70, 0, 100], 4, 4, 700, id='narrow_shared'),
    pytest.param([1] * 40, [64 + 7 * i for i in range(40)], 4, 1, 1300, id='wide_shared'),
    pytest.param([150, 40], [10, 250], 2, 1, 700, id='wide'),
    pytest.param([40], [1500], 2, 1, 0, id='wide_pieces'),
])
def test_attention_nan_and_infinite_scores(device, new, before, heads, kv_heads, prefix):
    """A key that makes a score NaN or +infinity makes NaN of every row that sees it;
    one that makes all of a row's scores but one -infinity leaves that row its
    one value; both in any piece of the list, in the middle of a tile."""
    c = Case(device, new, before, heads, kv_heads, prefix)
    c.q[:] = c.q.abs() + 0.5
    b, n = len(new) - 1, new[-1]
    at = before[-1] // 2
    row = 64 * int(c.table[b, at // 64]) + at % 64
    keep = c.k[0, row].clone()
    clean = tuple(x.clone() for x in c.attend())
    for value in (math.nan, math.inf):
        c.k[0, row, :, 7] = value
        out, lse = c.attend()
        assert torch.isnan(out[c.N - n:]).all()
        assert torch.equal(out[:c.N - n], clean[0][:c.N - n]) and torch.equal(lse[:c.N - n], clean[1][:c.N - n])
        c.k[0, row] = keep
    # every key that the last sequence sees but one at -infinity
    held = before[-1] + n
    rows = [64 * int(p) + r for i, p in enumerate(c.prefix.tolist()) for r in range(min(64, prefix - 64 * i))] + \
        [64 * int(c.table[b, i // 64]) + i % 64 for i in range(held)]
    c.k[0, rows, :, 7] = -math.inf
    c.k[0, row] = keep
    out, lse = c.attend()
    z = (c.q[c.N - n:].double().reshape(n, kv_heads, -1, 128) * c.k[0, row].double()[None, :, None]).sum(-1) * 128 ** -0.5
    want = c.v[0, row].double()[None, :, None].expand(n, kv_heads, heads // kv_heads, 128).reshape(n, heads, 128)
    u = torch.finfo(c.dtype).eps / 2
    assert ((out[c.N - n:].double() - want).abs() <= (2 * u + 2.0 ** -12) * want.abs()).all()
    assert ((lse[c.N - n:].double() - z.reshape(n, heads)).abs() <= 2.0 ** -13 + 2.0 ** -20).all()


def test_attention_layouts(device):
    """K and V side by side in one cache, head-major and broadcast queries, out in
    place of q, a table whose entries behind the sequence are garbage."""
    c = Case(device, [5, 40], [100, 3], 4, 2, 200, width=9)
    want, want_lse = c.attend()
    want, want_lse = want.clone(), want_lse.clone()
    both = torch.stack([c.k[0], c.v[0]], 1)[None]
    c.k, c.v = both[:, :, 0], both[:, :, 1]
    used = -(-c.lengths // 64)
    c.table[torch.arange(9, device=device) >= used[:, None]] = 0x7fffffff
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    got, lse = c.attend()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    got, lse = c.attend(out=c.q)
    assert got is c.q and torch.equal(got, want) and torch.equal(lse, want_lse)
    one = c.wide[:1, :1].expand(c.N, c.H, 128)
    c.q = one
    a = c.attend()[0].clone()
    c.q = one.contiguous()
    assert torch.equal(c.attend()[0], a)


def test_attention_no_rows_at_all(device):
    """Every sequence brings no token: nothing is written, in either form of
    call."""
    for new in ([0, 0, 0], [0]):
        c = Case(device, new, [70] * len(new), 2, 1, 90, padding=9)
        out = torch.full_like(c.q, 5.0)
        got, _ = c.attend(out=out)
        assert (got == 5.0).all()


def test_attention_many_ragged_sequences(device):
    """More sequences than a wave scans at once, empty ones among them."""
    new = [(7 * i) % 5 for i in range(150)]
    c = Case(device, new, [(13 * i) % 90 for i in range(150)], 2, 1, 33)
    c.check(*c.attend())


@pytest.mark.parametrize('count', [255, 257, 700])
def test_attention_more_sequences_than_a_pass_counts(device, count):
    """Tiles found among more than 256 sequences, runs of empty ones among them,
    on either side of a pass's end."""
    new = [0 if i % 9 < 4 or 250 < i < 256 else 1 + i % 3 for i in range(count)]
    new[-1] = 2
    c = Case(device, new, [(13 * i) % 70 for i in range(count)], 2, 1, 33)
    c.check(*c.attend())


def test_attention_in_place_and_two_threads(device):
    """Output rows over their own query rows, in narrow and wide tiles; two threads
    that call with different sizes at once, each on a stream of its own."""
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
    for c, (out, lse) in zip(cs, want):
        q = c.q.clone()
        c.q = q
        got, got_lse = c.attend(out=q)
        assert got is q and torch.equal(q, out) and torch.equal(got_lse, lse)


def test_attention_graphs_that_share_a_workspace(device):
    """Two captured calls of different sizes with one workspace, replayed in turn on
    one stream, between eager calls: each replay equals the eager call."""
    cs = [Case(device, [1] * 12, [50 * i for i in range(12)], 8, 2, 3000, seed=1),
          Case(device, [1] * 9, [30 * i for i in range(9)], 8, 2, 4000, seed=2)]
    ws, graphs, got = Workspace(), [], []
    want = [tuple(x.clone() for x in c.attend()) for c in cs]
    for c in cs:
        c.attend(ws=ws)
    torch.cuda.synchronize()
    for c in cs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(c.attend(ws=ws))
    for _ in range(3):
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
            cs[i].attend(ws=Workspace())
            torch.cuda.synchronize()


def test_attention_two_streams_at_once(device):
    """Two calls in flight together, each with a workspace of its own."""
    cs = [Case(device, [1] * 12, [50 * i for i in range(12)], 8, 2, 3000, seed=s) for s in (1, 2)]
    want = [tuple(x.clone() for x in c.attend()) for c in cs]
    torch.cuda.synchronize()
    streams, ws, got = [torch.cuda.Stream() for _ in cs], [Workspace() for _ in cs], [None, None]
    for _ in range(10):
        for i, c in enumerate(cs):
            with torch.cuda.stream(streams[i]):
                got[i] = c.attend(ws=ws[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_attention_workspace_of_many_sizes(device):
    """Calls of many sizes, as a server makes them, share a few buffers for their
    pieces."""
    ws = Workspace()
    for n in range(1, 25):
        c = Case(device, [1] * n, [40] * n, 4, 2, 600)
        c.check(*c.attend(ws=ws))
    sizes = [key[1][0] for key in ws.entries if key[0] == 'paged_part']
    assert sizes and len(sizes) <= 8 and all(x & (x - 1) == 0 for x in sizes)


def test_results_of_many_sizes_in_one_workspace(device):
    """Steps whose token count changes from call to call, their results in one
    workspace's shared buffers, the rotated queries passed on from there; a
    result turned again in place."""
    ws, f = Workspace(), freqs(device, 64)
    for n in (5, 8, 3, 9, 16, 1, 7):
        c = Case(device, [2] * n, [40] * n, 4, 2, 600)
        k, v = kv_parts(c)
        q = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, freqs=f, workspace=ws)
        want = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, freqs=f)
        assert torch.equal(q, want)
        c.q = q
        out, lse = c.attend(ws=ws)
        c.q = want
        c.check(out, lse)
        again = paged.append(k, v, c.k, c.v, c.table, c.held, q=q, freqs=f, workspace=ws)
        assert again.data_ptr() == q.data_ptr()
        assert torch.equal(again, paged.append(k, v, c.k, c.v, c.table, c.held, q=want, freqs=f))
    counts = [sum(key[0] == name for key in ws.entries) for name in ('paged_q', 'paged_out', 'paged_lse')]
    assert counts == [4, 4, 4]              # of 2, 8, 16 and 32 rows


def test_attention_sizes_that_no_grid_holds(device):
    """2^25 tiles of 256 threads are refused before anything is launched."""
    size = _lib.lib().ssa_paged_attention_workspace_bytes
    assert size(1 << 20, 1 << 20, 32, 32, 0, 1, 0, 1) == -1
    assert size(1 << 18, 1 << 18, 32, 32, 0, 1, 0, 1) >= 0


def append_case(device, c, k, v, **more):
    q = c.q
    ck, cv = c.k.clone(), c.v.clone()
    want = oracle.append(k, v, ck, cv, c.table, c.held, c.starts, q=q, **more)
    got = paged.append(k, v, c.k, c.v, c.table, c.held, q=q, starts=c.starts, **more)
    u = torch.finfo(c.dtype).eps / 2
    size = q.cpu().double().abs().max() + k.cpu().double().abs().max()
    assert ((got.cpu().double()[:c.N] - want[0][:c.N]).abs() <= u * want[0][:c.N].abs() + 2.0 ** -20 * size).all()
    touched = want[3]
    new_k, new_v = c.k[0].cpu(), c.v[0].cpu()
    d = (new_k[touched].double() - want[1][0, touched]).abs()
    assert (d <= u * want[1][0, touched].abs() + 2.0 ** -20 * size).all()
    assert torch.equal(new_v[touched].double(), want[2][0, touched])
    bits = torch.int16
    assert torch.equal(new_k[~touched].view(bits), ck[0].cpu()[~touched].view(bits))
    assert torch.equal(new_v[~touched].view(bits), cv[0].cpu()[~touched].view(bits))
    return got


def kv_parts(c, padding=0, seed=9):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(c.N + padding, 2 * c.G, 128, generator=g).to(c.dtype).to(c.device)
    return kv[:, :c.G], kv[:, c.G:]


def freqs(device, n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).to(device)


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
    append_case(device, c, *kv_parts(c), freqs=freqs(device, pairs), interleaved=interleaved, first=1234567)


def test_append_many_tokens(device):
    """Enough tokens for one wave each."""
    c = Case(device, [3000, 1200], [10, 0], 3, 1)
    append_case(device, c, *kv_parts(c), freqs=freqs(device, 64))


def test_append_more_sequences_than_a_wave_counts(device):
    """Tokens of 300 sequences, empty ones among them."""
    new = [0 if i % 5 < 2 else 1 + i % 2 for i in range(300)]
    c = Case(device, new, [(7 * i) % 100 for i in range(300)], 2, 1)
    append_case(device, c, *kv_parts(c), freqs=freqs(device, 64))


@pytest.mark.parametrize('pairs', [1, 7, 63])
def test_append_odd_pair_counts(device, pairs):
    c = Case(device, [9], [0], 2, 1)
    append_case(device, c, *kv_parts(c), freqs=freqs(device, pairs))


def test_append_axes_and_far_positions(device):
    """Three axes, positions of either sign up to the ends of int32: the angles
    hold to a float32 step."""
    c = Case(device, [40, 25], [0, 7], 4, 4)
    g = torch.Generator().manual_seed(4)
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (c.N, 3), generator=g).to(torch.int32).to(device)
    f = torch.cat([freqs(device, n) for n in (22, 21, 21)])
    append_case(device, c, *kv_parts(c), freqs=f, axes=(22, 21, 21), positions=pos)
    append_case(device, c, *kv_parts(c), freqs=f[:43], axes=(22, 21), positions=pos[:, :2].contiguous())
    append_case(device, c, *kv_parts(c), freqs=f, positions=pos[:, 0].contiguous())


def test_append_without_rotation_copies_bits(device):
    c = Case(device, [5, 66], [3, 0], 2, 2)
    k, v = kv_parts(c)
    k[0, 0, 0], k[1, 0, 1] = math.inf, -0.0
    got = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, starts=c.starts)
    assert torch.equal(got.view(torch.int16), c.q.contiguous().view(torch.int16))
    rows = [64 * int(c.table[0, 0]) + 3 + i for i in range(5)] + \
        [64 * int(c.table[1, i // 64]) + i % 64 for i in range(66)]
    for cache, new in ((c.k, k), (c.v, v)):
        assert torch.equal(cache[0, rows].view(torch.int16), new.contiguous().view(torch.int16))
    # the elements behind the pairs are copied, whatever they hold
    k[2, 0, 100] = math.nan
    paged.append(k, v, c.k, c.v, c.table, c.held, starts=c.starts, freqs=freqs(device, 40))
    row = 64 * int(c.table[0, 0]) + 3 + 2
    assert torch.isnan(c.k[0, row, 0, 100]) and torch.isfinite(c.k[0, row, 0].float()).sum() == 127


def test_append_outside_the_table_or_cache(device):
    """Tokens behind the table's end or on absent pages are not written, their
    queries still turn; padded rows are left alone."""
    c = Case(device, [4, 70], [60, 0], 2, 1, padding=5, width=2)
    used = c.table.flatten().tolist()
    c.table[1, 1] = -1
    c.table[0, 1] = [p for p in range(c.k.shape[1] // 64) if p not in used][0]
    c.held = ints([126, 0], device)
    k, v = kv_parts(c, padding=5)
    q_out = torch.full_like(c.q, 3.0)
    before = c.k.clone()
    want = oracle.append(k, v, c.k, c.v, c.table, c.held, c.starts, q=c.q, freqs=freqs(device, 64))
    got = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, q_out=q_out, starts=c.starts, freqs=freqs(device, 64))
    touched = want[3]
    assert int(touched.sum()) == 2 + 64
    assert torch.equal(c.k[0].cpu()[~touched].view(torch.int16), before[0].cpu()[~touched].view(torch.int16))
    assert (got[c.N:] == 3.0).all() and not (got[:c.N] == 3.0).all(-1).any()


def test_append_in_place_and_head_major(device):
    c = Case(device, [7], [60], 3, 2, head_major=True)
    k, v = kv_parts(c)
    plain = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, freqs=freqs(device, 48), interleaved=False)
    ck = c.k.clone()
    got = paged.append(k, v, c.k, c.v, c.table, c.held, q=c.q, q_out=c.q, freqs=freqs(device, 48), interleaved=False)
    assert got is c.q and torch.equal(plain, c.q)
    assert torch.equal(ck.contiguous().view(torch.int16), c.k.contiguous().view(torch.int16))


def test_cache_offsets_past_32_bits(device):
    """Pages beyond 2^31 elements (and 2^32 bytes) of a cache."""
    G, pages = 64, 4200                      # 64 x 128 elements a row: 2.2e9 elements
    k = torch.zeros(1, 64 * pages, G, 128, dtype=BF16, device=device)
    v = torch.zeros_like(k)
    table = ints([[pages - 1, 1], [pages - 2, pages - 3]], device)
    held, lengths = ints([3, 64], device), ints([5, 66], device)
    g = torch.Generator(device=device).manual_seed(1)
    rows = torch.randn(4, 3 * G, 128, generator=g, device=device).to(BF16)
    q, kk, vv = rows[:, :G], rows[:, G:2 * G], rows[:, 2 * G:]
    for x in (k, v):
        for pg in (pages - 1, pages - 2, pages - 3, pages - 4):
            x[0, 64 * pg:64 * pg + 64] = torch.randn(64, G, 128, generator=g, device=device).to(BF16)
    paged.append(kk, vv, k, v, table, held)
    assert torch.equal(k[0, 64 * (pages - 1) + 3:64 * (pages - 1) + 5], kk[:2])
    assert torch.equal(v[0, 64 * (pages - 3):64 * (pages - 3) + 2], vv[2:])
    prefix = ints([pages - 4], device)
    out = paged.attention(q, k, v, prefix, 50, table, lengths, Workspace())
    heads = [0, 63]
    small = [x[:, :, heads] for x in (k, v)]
    want, _, spread = oracle.attention(q[:, heads], small[0], small[1], prefix, 50, table, lengths,
                                       torch.tensor([0, 2, 4]))
    u = torch.finfo(BF16).eps / 2
    assert ((out[:, heads].cpu().double() - want).abs() <= u * want.abs() + (u + 2.0 ** -11) * spread + 2.0 ** -24).all()


def test_steps_of_several_sequences(device):
    """As they are used: a common prompt, then three sequences that append and
    attend token by token; equal to attention over the whole of each at once."""
    H, G, P, B, steps = 4, 2, 150, 3, 70
    c = Case(device, [0] * B, [0] * B, H, G, P, width=2, spare=2 * B)
    free = [p for p in range(c.k.shape[1] // 64) if p not in c.prefix.tolist()]
    c.table = ints([free[2 * b:2 * b + 2] for b in range(B)], device)
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(steps, B, H + 2 * G, 128, generator=g).to(BF16).to(device)
    f, ws = freqs(device, 64), Workspace()
    held = ints([0] * B, device)
    outs = []
    for s in range(steps):
        q, k, v = rows[s, :, :H], rows[s, :, H:H + G], rows[s, :, H + G:]
        q = paged.append(k, v, c.k, c.v, c.table, held, q=q, freqs=f, first=P, workspace=ws)
        held += 1
        outs.append(paged.attention(q, c.k, c.v, c.prefix, P, c.table, held, ws).clone())
    got = torch.stack(outs, 1).reshape(B * steps, H, 128)
    # the same at once, in an empty copy of the cache
    k2, v2 = c.k.clone(), c.v.clone()
    for b in range(B):
        for pg in c.table[b].tolist():
            k2[0, 64 * pg:64 * pg + 64] = math.nan
            v2[0, 64 * pg:64 * pg + 64] = math.nan
    flat = rows.transpose(0, 1).reshape(B * steps, H + 2 * G, 128)
    zero = ints([0] * B, device)
    q = paged.append(flat[:, H:H + G], flat[:, H + G:], k2, v2, c.table, zero, q=flat[:, :H], freqs=f, first=P)
    assert torch.equal(k2.view(torch.int16), c.k.view(torch.int16))
    out = paged.attention(q, k2, v2, c.prefix, P, c.table, held, Workspace())
    want, _, spread = oracle.attention(q, k2, v2, c.prefix, P, c.table, held, torch.arange(B + 1) * steps)
    u = torch.finfo(BF16).eps / 2
    for x in (got, out):
        assert ((x.cpu().double() - want).abs() <= u * want.abs() + (u + 2.0 ** -11) * spread + 2.0 ** -24).all()


def test_captured_step_replays_with_new_lengths(device):
    """An append and an attention captured in a graph and replayed token by token:
    lengths, rows and queries change on the device between replays; every
    replay equals the eager calls bit for bit."""
    c = Case(device, [1] * 6, [0, 5, 63, 64, 100, 126], 8, 2, 700, width=3)
    total = c.k.shape[1] // 64
    k = torch.randn(1, 64 * (total + 18), 2, 128, device=device).to(BF16)
    v = torch.randn(1, 64 * (total + 18), 2, 128, device=device).to(BF16)
    table = (total + torch.arange(18, device=device, dtype=torch.int32)).reshape(6, 3)
    rows = torch.empty(6, 12, 128, dtype=BF16, device=device)
    held, lengths = c.held.clone(), c.held + 1
    f = freqs(device, 64)

    def step(ws, k, v):
        q = paged.append(rows[:, 8:10], rows[:, 10:], k, v, table, held, q=rows[:, :8], freqs=f, first=700, workspace=ws)
        return paged.attention(q, k, v, c.prefix, 700, table, lengths, ws, want_lse=True)

    def fill(s):
        rows.copy_(torch.randn(6, 12, 128, generator=torch.Generator().manual_seed(s)).to(BF16))

    fill(0)
    ws, eager_ws = Workspace(), Workspace()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ws, k, v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(ws, k, v)
    eager_k, eager_v = k.clone(), v.clone()
    for s in range(1, 5):
        fill(s)
        held += 13
        lengths.copy_(held + 1)
        ws.tensor('paged_part', ws_shape(ws), device, torch.uint8).fill_(255)    # any contents will do
        torch.randn(1 << 20, device=device).sum()
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = step(eager_ws, eager_k, eager_v)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert torch.equal(k, eager_k) and torch.equal(v, eager_v)


def ws_shape(ws):
    shapes = [key[1] for key in ws.entries if key[0] == 'paged_part']
    return shapes[0] if shapes else (16,)


def test_other_stream(device):
    c = Case(device, [1] * 4, [100, 10, 64, 0], 4, 2, 300)
    want, want_lse = c.attend()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, lse = c.attend()
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
