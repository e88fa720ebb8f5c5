"""Attention with shaped scores (a cap, slopes, a window) over the 16-bit and the
8-bit paged cache, against float64.

Tolerances as for plain scores (see test_gpu_paged8.py): the output's rounding, a
probability's rounding, a score's error, float32 sums.  A cap adds at most 2^-22
of itself to a score's error, a slope the roundings of its product and its sum,
2^-22 of the largest fall among the keys that are seen; both are absolute errors
of a score and so relative ones of a probability.  The spread that they are
measured by is sum p |v| / sum p."""
import math

import pytest
import torch

from oracle import paged8 as oracle
from streaming_sparse_amd import paged, paged8
from streaming_sparse_amd.attention import Workspace
from test_gpu_paged8 import BF16, FP16, SHAPES, Case, ints

pytestmark = pytest.mark.gpu


def slopes_of(heads, device, top=0.5):
    return top * torch.exp2(-8.0 * torch.arange(heads, device=device) / heads)


class Shaped(Case):
    """A Case whose rows lie in a cache of either kind, the same values in both."""

    def __init__(self, bits, *args, **more):
        super().__init__(*args, **more)
        self.bits = bits

    def sixteen(self):
        k, v = (x.to(self.dtype) for x in oracle.pages8(self.cache))
        return [x.transpose(1, 2).reshape(1, -1, self.G, 128).contiguous() for x in (k, v)]

    def attend(self, causal=True, ragged=True, ws=None, **more):
        if self.bits == 8:
            return super().attend(causal, ragged, ws, **more)
        return paged.attention(self.q, *self.sixteen(), self.prefix, self.P, self.table, self.lengths, ws or Workspace(),
                               starts=self.starts if ragged else None, causal=causal, want_lse=True, **more)

    def check_shaped(self, out, lse, causal=True, cap=None, slopes=None, window=None, **more):
        fall = 0.0 if slopes is None else float(slopes.abs().max()) * (self.P + max(self.lengths.tolist()) + 1)
        score = 2.0 ** -13 + (cap or 0.0) * 2.0 ** -22 + min(fall, 2.0 ** 12) * 2.0 ** -22 + more.pop('sums', 0.0)
        self.check(out, lse, causal, score=score, cap=cap, slopes=slopes, window=window, **more)


HOW = [
    pytest.param(dict(cap=5.0), id='cap'),
    pytest.param(dict(slopes=True), id='slopes'),
    pytest.param(dict(window=70), id='window'),
    pytest.param(dict(cap=30.0, slopes=True, window=33), id='all'),
]


def given(how, heads, device):
    return {**how, **({'slopes': slopes_of(heads, device)} if how.get('slopes') else {})}


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('causal', [True, False], ids=['causal', 'full'])
@pytest.mark.parametrize('how', HOW)
@pytest.mark.parametrize('new,before,heads,kv_heads,prefix', SHAPES)
def test_shaped(device, new, before, heads, kv_heads, prefix, how, causal, bits):
    c = Shaped(bits, device, new, before, heads, kv_heads, prefix, BF16 if causal else FP16)
    how = given(how, heads, device)
    c.check_shaped(*c.attend(causal, **how), causal, **how)


LARGE = [
    # every way through the kernels
    pytest.param(8, 1, 200, 8, 8, 9000, True, BF16, dict(cap=20.0, slopes=True), id='apart_narrow'),
    pytest.param(9, 1, 5000, 3, 1, 500, True, FP16, dict(window=1000), id='narrow_pieces'),
    pytest.param(1, 1, 30000, 8, 2, 70, True, BF16, dict(cap=50.0, window=20000), id='narrow_many_pieces'),
    pytest.param(40, 3, 400, 12, 12, 0, True, FP16, dict(slopes=True, window=100), id='narrow_whole'),
    pytest.param(12, 1, 700, 8, 2, 9000, True, BF16, dict(cap=50.0, slopes=True, window=300), id='apart_48_rows'),
    pytest.param(90, 1, 700, 6, 2, 20000, True, BF16, dict(cap=50.0, slopes=True), id='apart_wide_many_pieces'),
    pytest.param(30, 7, 1900, 14, 2, 700, True, FP16, dict(slopes=True, window=300), id='wide_few_tokens'),
    pytest.param(300, 1, 330, 16, 8, 700, True, BF16, dict(window=65), id='apart_items_in_turn'),
    pytest.param(1, 200, 50, 8, 2, 30000, True, BF16, dict(cap=30.0, window=64), id='wide_many_pieces'),
    pytest.param(3, 601, 7, 8, 8, 126, True, FP16, dict(window=200, cap=5.0), id='half_wide_whole'),
    pytest.param(1, 1265, 1340, 12, 4, 248, True, BF16, dict(window=500), id='half_wide_window'),
    pytest.param(2, 700, 0, 48, 48, 1000, False, BF16, dict(cap=50.0), id='wide_rounds'),
    pytest.param(1, 2000, 100, 12, 12, 10, True, BF16, dict(slopes=True), id='causal_cut'),
    pytest.param(1, 2000, 1000, 12, 12, 10, True, BF16, dict(window=900, cap=30.0), id='causal_window'),
    pytest.param(5, 530, 1600, 8, 1, 4300, False, BF16, dict(slopes=True, window=700), id='prompts'),
]


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('batch,new,held,heads,kv_heads,prefix,causal,dtype,how', LARGE)
def test_shaped_large(device, batch, new, held, heads, kv_heads, prefix, causal, dtype, how, bits):
    before = torch.randint(0, held + 1, (batch,), generator=torch.Generator().manual_seed(4)).tolist()
    before[0] = held
    c = Shaped(bits, device, [new] * batch, before, heads, kv_heads, prefix, dtype)
    how = given(how, heads, device)
    ws = Workspace()
    out, lse = (x.clone() for x in c.attend(causal, ragged=False, ws=ws, **how))
    # a lane adds up to 16384 of its row's probabilities one by one
    c.check_shaped(out, lse, causal, sums=2.0 ** -10, **how)
    again = c.attend(causal, ragged=False, ws=ws, **how)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for parts in (True, False):
        c.check_shaped(*c.attend(causal, single_av=parts, **how), causal, sums=2.0 ** -10, **how)


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('new,before,heads,kv_heads,window', [
    pytest.param([1], [1000], 4, 2, 100, id='step'),
    pytest.param([1] * 50, [40 * i for i in range(50)], 4, 1, 130, id='steps'),
    pytest.param([5, 0, 9], [900, 500, 64], 2, 2, 64, id='few'),
    pytest.param([200, 90], [700, 0], 4, 2, 150, id='prompts'),
    pytest.param([300], [2000], 2, 2, 1, id='itself_alone'),
])
def test_window_over_released_pages(device, new, before, heads, kv_heads, window, bits):
    """Pages that have left every window are gone from the table; in the first page that
    is still seen, and in the released ones, the rows before the window hold NaN."""
    c = Shaped(bits, device, new, before, heads, kv_heads, 100)
    table = c.table.clone()
    for b, n in enumerate(before):
        low = max(n - window + 1, 0)
        for at in range(low):
            page = int(table[b, at // 64])
            for x in (c.cache.k, c.cache.v):
                x.view(torch.uint8)[page, :, at % 64] = 0x7f
        if low // 64:
            c.table[b, :low // 64] = -1
    for causal in (True, False):
        c.check_shaped(*c.attend(causal, window=window), causal, window=window)


@pytest.mark.parametrize('bits', [16, 8])
def test_windows_of_every_size_about_a_page(device, bits):
    c = Shaped(bits, device, [3, 70], [200, 61], 2, 1, 30)
    for window in (1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1 << 20, (1 << 30) - 1):
        c.check_shaped(*c.attend(window=window), window=window)
    a = [x.clone() for x in c.attend(window=1 << 40)]
    b = c.attend(window=(1 << 30) - 1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize('bits', [16, 8])
def test_shape_that_changes_nothing(device, bits):
    """Slopes of zero and a window that nothing falls out of: plain attention, up to its
    roundings; a cap far above the scores too, up to 2^-22 of it."""
    for new in ([1, 1], [150]):
        c = Shaped(bits, device, new, [200] * len(new), 2, 2, 300)
        for how in (dict(slopes=torch.zeros(2, device=device)), dict(window=10 ** 6), dict(cap=500.0)):
            out, lse = c.attend(**how)
            if 'cap' not in how:
                c.check_shaped(out, lse)
            c.check_shaped(out, lse, **how)


@pytest.mark.parametrize('bits', [16, 8])
def test_negative_slopes_and_large_falls(device, bits):
    """Far keys above near ones; falls of thousands, under which one key is left."""
    for new, ragged in (([1, 1, 1], False), ([2, 0, 160], True)):
        c = Shaped(bits, device, new, [300, 20, 77], 4, 2, 500)
        for slopes in ([-0.01, 0.02, 0.0, -0.003], [50.0, 3.0, 0.7, 10.0]):
            slopes = torch.tensor(slopes, device=device)
            for causal in (True, False):
                c.check_shaped(*c.attend(causal, ragged, slopes=slopes), causal, slopes=slopes)


@pytest.mark.parametrize('bits', [16, 8])
def test_cap_under_large_scores(device, bits):
    """Scores many times the cap, of both signs: all of a row's probabilities come from
    the tanh's ends."""
    for new in ([1], [130]):
        c = Shaped(bits, device, new, [400], 2, 1, 200)
        c.check_shaped(*c.attend(cap=3.0, scale=40.0), cap=3.0, scale=40.0)


@pytest.mark.parametrize('bits', [16, 8])
def test_shaped_rows_that_see_nothing(device, bits):
    for new in ([6, 2], [200, 3]):
        c = Shaped(bits, device, new, [0, 0], 2, 1, 0)
        c.lengths = ints([4, 0], device)
        how = dict(cap=5.0, slopes=slopes_of(2, device), window=2)
        out, lse = c.attend(**how)
        c.check_shaped(out, lse, **how)
        assert (out[:new[0] - 4] == 0).all() and torch.isinf(lse[:new[0] - 4]).all()


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('causal', [True, False], ids=['causal', 'full'])
def test_shaped_lengths_past_the_table(device, causal, bits):
    for new, before, drop in (([4], [126], 1), ([1] * 40, [64 + 7 * i for i in range(40)], 3), ([300, 40], [10, 250], 2)):
        c = Shaped(bits, device, new, before, 2, 1, 70)
        c.table = c.table[:, :max(1, c.table.shape[1] - drop)].contiguous()
        how = dict(slopes=slopes_of(2, device), window=90)
        c.check_shaped(*c.attend(causal, **how), causal, **how)


@pytest.mark.parametrize('bits', [16, 8])
def test_shaped_nan_shows(device, bits):
    """A NaN key reaches the rows that see it, through a cap too, and no row whose window
    it has left."""
    c = Shaped(bits, device, [1, 1], [100, 100], 2, 1, 100)
    c.cache.k.view(torch.uint8)[int(c.table[0, 0]), 0, 5, 3] = 0x7f
    out, _ = c.attend(cap=5.0)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    out, lse = c.attend(cap=5.0, window=95)
    c.check_shaped(out, lse, cap=5.0, window=95)


@pytest.mark.parametrize('bits', [16, 8])
def test_shaped_captured_step(device, bits):
    """A step captured in a graph, replayed as the sequences grow, eager work between."""
    c = Shaped(bits, device, [1] * 6, [130, 5, 63, 64, 100, 126], 8, 2, 300)
    how = dict(cap=20.0, slopes=slopes_of(8, device), window=70)
    lengths = c.lengths.clone()
    k, v = c.sixteen()
    ws = Workspace()

    def step(ws):
        if bits == 8:
            return paged8.attention(c.q, c.cache, c.prefix, 300, c.table, lengths, ws, want_lse=True, **how)
        return paged.attention(c.q, k, v, c.prefix, 300, c.table, lengths, ws, want_lse=True, **how)

    step(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(ws)
    for less in (3, 0, 5, 1):
        lengths.copy_((c.lengths - less).clamp_min(1))
        torch.randn(1 << 20, device=device).sum()
        graph.replay()
        torch.cuda.synchronize()
        want = step(Workspace())
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        keep, c.lengths = c.lengths, lengths
        c.check_shaped(*want, **how)
        c.lengths = keep


def test_both_caches_give_the_same(device):
    """The same values in 16 and in 8 bits: the same outputs, up to both sides' roundings."""
    how = dict(cap=20.0, slopes=slopes_of(4, device), window=200)
    for new, before in (([1] * 6, [300] * 6), ([90, 40], [20, 130])):
        a, b = (Shaped(bits, device, new, before, 4, 2, 150) for bits in (8, 16))
        x, y = a.attend(**how), b.attend(**how)
        size = float(b.sixteen()[1].nan_to_num().abs().max())
        u = torch.finfo(BF16).eps / 2
        assert ((x[0].double() - y[0].double()).abs() <= 2 * u * y[0].double().abs() + (2 * u + 2.0 ** -11) * size).all()
        assert ((x[1] - y[1]).abs() <= 2.0 ** -11).all() and math.isfinite(size)
