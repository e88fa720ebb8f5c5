"""What the 8-bit paged cache's arithmetic may lose, where a looser bound would hide it.

u = finfo(dtype).eps / 2 is half a step of the output type, 2^-11 half a step of the
fp16 part that stands for two bf16 ones."""
import pytest
import torch

from oracle import paged8 as oracle
from streaming_sparse_amd import paged8
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize('shaped', [False, True], ids=['plain', 'shaped'])
@pytest.mark.parametrize('gap', [15, 8, 0])
@pytest.mark.parametrize('below', [14.0, 16.5, 17.0, 18.0])
@pytest.mark.parametrize('batch,new,single', [
    pytest.param(64, 1, None, id='narrow'),
    pytest.param(1, 40, False, id='wide'),
])
def test_many_small_probabilities_keep_their_weight(device, batch, new, single, below, gap, shaped):
    """Thousands of keys whose probabilities are 2^-14 to 2^-18 of a dominant one's, and whose values' powers of two lie
    `gap` below that of a row without weight that comes first.  All values are alike in size and sign, so that a
    probability that loses bits shows in the output: by up to 4096 * 2^-17, 3% of it.  The scores' products and sums are
    exact, a probability is off by 2^-20 for its exponential and 2^-11 for its part, sums of 2^12 terms by 2^-12."""
    G, pages = 8, 256
    g = torch.Generator(device=device).manual_seed(1)
    cache = paged8.Cache.empty(pages, G, device)
    cache.scales.fill_(120)
    v = 256 + 192 * torch.rand(G, 1, 128, generator=g, device=device)
    cache.v.copy_(v.expand(pages, G, 64, 128).to(torch.float8_e4m3fn))
    k = torch.full((pages, G, 64, 128), -64.0, device=device)          # with 2^-7: -0.5
    for w in range(4):                                                  # a narrow tile's waves take pages w, w + 4, ...
        k[w, :, 0] = -448.0
        k[w, :, 1] = 64.0
        cache.scales[w, :, 1, 0] = 120 + gap
    cache.k.copy_(k.to(torch.float8_e4m3fn))
    q = torch.ones(batch * new, G, 128, device=device, dtype=BF16)
    # a key's score is +-64 scale: the dominant one's lies 128 scale log2(e) above the others'
    scale = below / (128 * 1.4426950408889634)
    table = torch.arange(pages, dtype=torch.int32, device=device).expand(batch, pages).contiguous()
    lengths = ints([64 * pages] * batch, device)
    shape = dict(window=1 << 20) if shaped else {}
    out = paged8.attention(q, cache, None, 0, table, lengths, Workspace(), causal=False, scale=scale, single_av=single, **shape)
    want, _, spread = oracle.attention(q[:new], *oracle.pages8(cache), None, 0, table[:1], lengths[:1], ints([0, new], device),
                                       causal=False, scale=scale)
    far = (out.double().unflatten(0, (batch, new)) - want).abs() / spread
    limit = torch.finfo(BF16).eps / 2 + 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -20
    assert float(far.max()) <= limit, (float(far.max()), limit)


@pytest.mark.parametrize('how', [dict(), dict(window=1 << 20)], ids=['plain', 'shaped'])
@pytest.mark.parametrize('batch,new,prefix,held', [
    pytest.param(64, 1, 0, 5, id='narrow'),
    pytest.param(1, 100, 0, 6, id='wide'),
    pytest.param(90, 1, 1500, 3, id='apart'),
])
def test_two_parts_that_are_asked_for(device, batch, new, prefix, held, how):
    """single_av=False: how many outputs are not the float64 result's rounding.  With all values of one sign an error e of
    an output, relative, takes |e| / step of them, step 2^-7 to 2^-8, to the other side of a border: of a few keys whose
    probabilities are off by 2^-16 / sqrt(12) each (two parts of 8 bits), scores by 2^-18 and exponentials by 2^-20,
    0.8 * 2^-17 / 2^-7.5, one in 900.  One fp16 part is off by 2^-10 / sqrt(12), the root of the sum of the squared
    probabilities of a few keys a half of that: one in 50.  At most one in 256 is allowed."""
    G, H = 8, 32
    width, shared = 2, -(-prefix // 64)
    pages = shared + batch * width
    g = torch.Generator(device=device).manual_seed(2)
    cache = paged8.Cache.empty(pages, G, device)
    v = 256 + 192 * torch.rand(pages, G, 64, 128, generator=g, device=device)
    cache.v.copy_(v.to(torch.float8_e4m3fn))
    k = torch.randn(pages, G, 64, 128, generator=g, device=device)
    k *= 64.0
    if shared:                            # all but two keys of the prefix's first two pages score about -40
        none = torch.ones(shared, 1, 64, 1, dtype=torch.bool, device=device)
        none[:2, :, 7:9] = False
        k[:shared, ..., :4] = torch.where(none, -448.0, k[:shared, ..., :4])
    cache.k.copy_(k.clamp(-448, 448).to(torch.float8_e4m3fn))
    cache.scales[:, :, 0] = 121
    cache.scales[:, :, 1] = torch.randint(116, 122, (pages, G, 64), generator=g, device=device).to(torch.uint8)
    q = torch.randn(batch * new, H, 128, generator=g, device=device).to(BF16)
    if shared:
        q[..., :4] = 16.0
    order = torch.arange(pages, dtype=torch.int32, device=device)
    table = order[shared:].reshape(batch, width).contiguous()
    lengths = ints([held] * batch, device)
    starts = torch.arange(batch + 1, device=device) * new
    out = paged8.attention(q, cache, order[:shared].contiguous(), prefix, table, lengths, Workspace(), causal=False,
                           single_av=False, **how)
    want, _, _ = oracle.attention(q, *oracle.pages8(cache), order[:shared], prefix, table, lengths, starts, causal=False)
    off = float((out != want.float().to(BF16)).double().mean())
    assert off <= 2.0 ** -8, off


WAYS = [
    # batch, new tokens, prefix, held
    pytest.param(64, 1, 0, 700, id='narrow'),
    pytest.param(90, 1, 1500, 70, id='apart'),
    pytest.param(8, 1, 3000, 70, id='narrow_apart'),
]


def case(device, batch, new, prefix, held, G=8, H=32):
    width, shared = -(-(held + new) // 64), -(-prefix // 64)
    pages = shared + batch * width
    g = torch.Generator(device=device).manual_seed(5)
    cache = paged8.Cache.empty(pages, G, device)
    for x in (cache.k, cache.v):
        x.copy_((100 * torch.randn(pages, G, 64, 128, generator=g, device=device)).clamp(-448, 448).to(torch.float8_e4m3fn))
    cache.scales.fill_(120)
    q = torch.randn(batch * new, H, 128, generator=g, device=device).to(BF16)
    order = torch.arange(pages, dtype=torch.int32, device=device)
    return cache, (q, cache, order[:shared].contiguous(), prefix, order[shared:].reshape(batch, width).contiguous(),
                   ints([held + new] * batch, device))


@pytest.mark.parametrize('how', [dict(), dict(window=1 << 20)], ids=['plain', 'shaped'])
@pytest.mark.parametrize('batch,new,prefix,held', WAYS)
def test_zero_rows_cost_no_part(device, batch, new, prefix, held, how):
    """A value row of zeros has the least power of two; the same outputs, bit for bit, as with its neighbours' power.
    One of NaN has it too, and shows."""
    cache, a = case(device, batch, new, prefix, held)
    cache.v.view(torch.uint8)[:, :, 5] = 0
    cache.v.view(torch.uint8)[::3, :, 11] = 0x80
    want = paged8.attention(*a, Workspace(), **how)
    cache.scales[:, :, 1, 5] = 1
    cache.scales[::3, :, 1, 11] = 1
    assert torch.equal(paged8.attention(*a, Workspace(), **how), want)
    exact = paged8.attention(*a, Workspace(), single_av=False, **how)
    assert not torch.equal(exact, want)              # so the comparison above tells one part from two
    page = int(a[4][0, 0])
    cache.v.view(torch.uint8)[page, 0, 5, 3] = 0x7f
    got = paged8.attention(*a, Workspace(), **how)
    assert torch.isnan(got[0, :4, 3]).all() and torch.isfinite(got[0, :4, 4:]).all() and torch.isfinite(got[1:]).all()
