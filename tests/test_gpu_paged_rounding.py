"""The size of the attention's errors, not only their bound: over a head and over
a call, the sum of their squares is that of the outputs' own rounding where a
probability meets V in two 16-bit parts, and that with a probability's rounding
where it meets V in one (oracle.paged.error_limit, with the derivation).  Sizes
that take every way through the kernels; a page or half page of V that is
left out or misplaced passes the limit several times."""
import math

import pytest
import torch

from oracle import paged as oracle
from streaming_sparse_amd import paged
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

CASES = [
    # batch, new tokens, equal, held, heads, K/V heads, prefix, causal, dtype, parts by default
    pytest.param(8, 1, True, 200, 8, 8, 9000, True, BF16, 2, id='apart_narrow'),
    pytest.param(9, 1, True, 200, 3, 1, 5000, True, FP16, 2, id='joint_narrow_pieces'),
    pytest.param(1, 1, True, 30, 8, 2, 30250, True, BF16, 2, id='joint_narrow_many_pieces'),
    pytest.param(40, 3, True, 400, 12, 12, 0, True, BF16, 2, id='joint_narrow_whole'),
    pytest.param(90, 1, True, 700, 6, 2, 20000, True, BF16, 2, id='apart_wide_many_pieces'),
    pytest.param(64, 1, True, 600, 16, 4, 16384, True, FP16, 2, id='apart_wide_steps'),
    pytest.param(30, 7, True, 90, 14, 2, 700, True, FP16, 1, id='joint_wide_few_tokens'),
    pytest.param(24, 5, True, 333, 28, 4, 5003, True, FP16, 1, id='apart_wide_more_rows'),
    pytest.param(300, 1, True, 130, 16, 8, 700, True, BF16, 2, id='apart_items_in_turn'),
    pytest.param(1, 200, True, 50, 8, 2, 30000, True, BF16, 1, id='joint_wide_many_pieces'),
    pytest.param(20, 64, True, 900, 12, 12, 0, True, FP16, 1, id='joint_wide_few_rows'),
    pytest.param(3, 601, True, 7, 8, 8, 126, True, FP16, 1, id='half_wide_whole'),
    pytest.param(1, 1265, True, 134, 12, 4, 248, True, BF16, 1, id='half_wide_causal_cut'),
    pytest.param(2, 700, True, 0, 48, 48, 1000, False, BF16, 1, id='joint_wide_rounds'),
    pytest.param(1, 2000, True, 100, 12, 12, 10, True, FP16, 1, id='causal_cut'),
    pytest.param(5, 530, False, 1600, 8, 1, 4300, False, BF16, 1, id='ragged_prompts'),
]


@pytest.mark.parametrize('batch,new,equal,held,heads,kv_heads,prefix,causal,dtype,parts', CASES)
def test_attention_rounds_as_it_says(device, batch, new, equal, held, heads, kv_heads, prefix, causal, dtype, parts):
    g = torch.Generator(device=device).manual_seed(batch + new)
    counts = torch.full((batch,), new) if equal else torch.randint(0, new + 1, (batch,),
                                                                   generator=torch.Generator().manual_seed(3))
    counts[-1] = new
    before = torch.randint(0, held + 1, (batch,), generator=torch.Generator().manual_seed(4))
    n, r = int(counts.sum()), heads // kv_heads
    shared, width = -(-prefix // 64), -(-int((counts + before).max()) // 64)
    pages = shared + batch * width
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    ids, table = order[:shared].contiguous(), order[shared:].reshape(batch, width).contiguous()
    k, v = (torch.randn(1, 64 * pages, kv_heads, 128, generator=g, device=device).to(dtype) for _ in range(2))
    q = torch.randn(n, heads, 128, generator=g, device=device).to(dtype)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32).to(device)
    lengths = (counts + before).to(torch.int32).to(device)
    got = {single: paged.attention(q, k, v, ids, prefix, table, lengths, Workspace(), causal=causal,
                                   starts=None if equal else starts, single_av=single).double()
           for single in (None, False, True)}

    want = torch.zeros(n, heads, 128, dtype=torch.float64, device=device)
    p2, p2v2 = torch.zeros(n, heads, dtype=torch.float64, device=device), torch.zeros_like(want)
    kp, vp = (x[0].view(-1, 64, kv_heads, 128) for x in (k, v))
    lo = starts.tolist()
    for b in range(batch):
        m, length = int(counts[b]), int(lengths[b])
        own = table[b, :-(-length // 64)].long()
        kk, vv = (torch.cat([x[ids.long()].reshape(-1, kv_heads, 128)[:prefix],
                             x[own].reshape(-1, kv_heads, 128)[:length]]).double() for x in (kp, vp))
        last = prefix + (length - m + torch.arange(m, device=device) if causal else
                         torch.full((m,), length - 1, device=device))
        hidden = torch.arange(len(kk), device=device) > last[:, None]
        for h in range(heads):
            z = (q[lo[b]:lo[b + 1], h].double() @ kk[:, h // r].t() * 128 ** -0.5).masked_fill(hidden, -math.inf)
            p = z.softmax(-1)
            at = slice(lo[b], lo[b + 1])
            want[at, h], p2[at, h], p2v2[at, h] = p @ vv[:, h // r], (p * p).sum(-1), (p * p) @ vv[:, h // r] ** 2

    # narrow tiles have two parts whatever is asked for
    narrow = n * r <= 32 * batch and (prefix == 0 or n * r <= 32 or batch == 1)
    for single, count in ((None, parts), (False, 2), (True, 2 if narrow else 1)):
        for h in range(heads):
            far = float((got[single][:, h] - want[:, h]).norm())
            limit = float(oracle.error_limit(want[:, h], p2[:, h], p2v2[:, h], dtype, count))
            assert far <= limit, (single, h, far, limit)
        far, limit = float((got[single] - want).norm()), float(oracle.error_limit(want, p2, p2v2, dtype, count))
        print(f'single_av={single}: {far / float(want.norm()):.3g} of the outputs, limit {limit / float(want.norm()):.3g}')
        assert far <= limit, (single, far, limit)
