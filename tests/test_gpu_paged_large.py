"""Shared-prefix attention at sizes that take every way through the kernels: tiles
of 32 and of 256 rows, the prefix apart or in one list with the sequence's
pages, lists whole and in few or many pieces, full rounds with a cut remainder,
causal prompts cut at one length.  Against float64 on the device.

Tolerances, with u = finfo(dtype).eps / 2: the output's rounding u |out|; a
probability's rounding to 16 bits at most u sum p |v| / sum p; a score's error
below 2^-13 (128 x 2^-24 sum |q k| scale, sum |q k| scale < 16); the float32 sums
over at most 32768 keys: a lane adds at most 16384 of them one by one, relative
error below 16384 x 2^-24 = 2^-10."""
import math

import pytest
import torch

from streaming_sparse_amd import paged
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

CASES = [
    # batch, new tokens, equal, held, heads, K/V heads, prefix, causal, dtype
    pytest.param(8, 1, True, 200, 8, 8, 9000, True, BF16, id='apart_narrow'),
    pytest.param(9, 1, True, 200, 3, 1, 5000, True, BF16, id='joint_narrow_pieces'),
    pytest.param(90, 1, True, 700, 6, 2, 20000, True, BF16, id='apart_wide_many_pieces'),
    pytest.param(30, 7, True, 90, 14, 2, 700, True, FP16, id='apart_wide_few_pieces'),
    pytest.param(12, 41, False, 300, 8, 8, 1500, True, BF16, id='apart_ragged'),
    pytest.param(300, 1, True, 130, 16, 8, 700, True, BF16, id='apart_items_in_turn'),
    pytest.param(200, 3, False, 500, 12, 12, 300, False, FP16, id='apart_ragged_items_in_turn'),
    pytest.param(1, 1, True, 30, 8, 2, 30000, True, FP16, id='joint_narrow_many_pieces'),
    pytest.param(40, 3, True, 400, 12, 12, 0, True, BF16, id='joint_narrow_whole'),
    pytest.param(1, 200, True, 50, 8, 2, 30000, True, BF16, id='joint_wide_many_pieces'),
    pytest.param(20, 64, True, 900, 12, 12, 0, True, FP16, id='joint_wide_few_rows'),
    pytest.param(3, 150, False, 700, 2, 1, 5, False, BF16, id='joint_wide_one_or_two_tiles'),
    pytest.param(3, 601, True, 7, 8, 8, 126, True, FP16, id='half_wide_whole'),
    pytest.param(1, 1265, True, 134, 12, 4, 248, True, BF16, id='half_wide_causal_cut'),
    pytest.param(2, 185, False, 725, 12, 3, 15, False, BF16, id='half_wide_pieces'),
    pytest.param(2, 700, True, 0, 48, 48, 1000, False, BF16, id='joint_wide_rounds'),
    pytest.param(1, 2000, True, 100, 12, 12, 10, True, BF16, id='causal_cut'),
    pytest.param(3, 1500, False, 10, 24, 24, 3, True, FP16, id='causal_whole'),
    pytest.param(5, 530, False, 1600, 8, 1, 4300, False, BF16, id='ragged_prompts'),
    pytest.param(2, 65, True, 0, 128, 1, 129, True, BF16, id='one_kv_head'),
]


@pytest.mark.parametrize('batch,new,equal,held,heads,kv_heads,prefix,causal,dtype', CASES)
def test_attention_large(device, batch, new, equal, held, heads, kv_heads, prefix, causal, dtype):
    g = torch.Generator(device=device).manual_seed(batch + new)
    counts = torch.full((batch,), new) if equal else torch.randint(0, new + 1, (batch,),
                                                                   generator=torch.Generator().manual_seed(3))
    counts[-1] = new
    before = torch.randint(0, held + 1, (batch,), generator=torch.Generator().manual_seed(4))
    n = int(counts.sum())
    shared, width = -(-prefix // 64), -(-int((counts + before).max()) // 64)
    pages = shared + batch * width
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    ids, table = order[:shared].contiguous(), order[shared:].reshape(batch, width).contiguous()
    k, v = (torch.randn(1, 64 * pages, kv_heads, 128, generator=g, device=device).to(dtype) for _ in range(2))
    q = torch.randn(n, heads, 128, generator=g, device=device).to(dtype)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32).to(device)
    lengths = (counts + before).to(torch.int32).to(device)
    ws = Workspace()
    out, lse = paged.attention(q, k, v, ids, prefix, table, lengths, ws, starts=None if equal else starts,
                               causal=causal, want_lse=True)
    out, lse = out.clone(), lse.clone()
    again = paged.attention(q, k, v, ids, prefix, table, lengths, ws, starts=None if equal else starts, causal=causal,
                            want_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])

    u, r = torch.finfo(dtype).eps / 2, heads // kv_heads
    kp, vp = (x[0].view(-1, 64, kv_heads, 128) for x in (k, v))
    lo = starts.tolist()
    for b in range(batch):
        m, length = int(counts[b]), int(lengths[b])
        if m == 0:
            continue
        own = table[b, :-(-length // 64)].long()
        kk, vv = (torch.cat([x[ids.long()].reshape(-1, kv_heads, 128)[:prefix],
                             x[own].reshape(-1, kv_heads, 128)[:length]]).double() for x in (kp, vp))
        last = prefix + (length - m + torch.arange(m, device=device) if causal else
                         torch.full((m,), length - 1, device=device))
        hidden = torch.arange(len(kk), device=device) > last[:, None]
        for h in range(heads):
            z = (q[lo[b]:lo[b + 1], h].double() @ kk[:, h // r].t() * 128 ** -0.5).masked_fill(hidden, -math.inf)
            p = z.softmax(-1)
            want, spread = p @ vv[:, h // r], p @ vv[:, h // r].abs()
            got = out[lo[b]:lo[b + 1], h].double()
            far = (got - want).abs() - (u * want.abs() + (u + 2.0 ** -13 + 2.0 ** -10) * spread + 2.0 ** -24)
            assert far.max() <= 0, (b, h, float(far.max()))
            off = (lse[lo[b]:lo[b + 1], h].double() - z.logsumexp(-1)).abs()
            assert off.max() <= 2.0 ** -13 + 2.0 ** -10 + 2.0 ** -18, (b, h, float(off.max()))
