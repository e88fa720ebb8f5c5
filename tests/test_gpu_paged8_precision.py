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
