"""The size of the errors of attention over 8-bit rows, and with shaped scores over either
cache, as test_gpu_paged_rounding has it for plain scores over 16-bit rows: over a
head and over a call, the sum of their squares is that of the outputs' own rounding
and of the parts in which a probability meets V (oracle.paged.error_limit).  Where one
fp16 part may stand for two bf16 ones, that one's.  A lost second part, or a page or
half page of V left out or misplaced, passes the limit.

Shaped scores add to the errors that are allowed for as 2^-15: a cap of 20 at most 2^-22
of itself to a score, 2^-17.7, a slope 2^-23 of a fall, 2^-18 where a key has weight
(falls below 32); with those named there 2^-15.5 together."""
import math

import pytest
import torch

from oracle import paged as limits
from oracle import paged8 as oracle
from streaming_sparse_amd import paged, paged8
from streaming_sparse_amd.attention import Workspace

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


class Call:
    """Sequences over 8-bit rows, pages anywhere; value rows' powers of two within 2^-3 .. 2^3, or, with `apart`, within
    2^-15 .. 2^15 from one row to the next (2^-7 .. 2^7 in fp16)."""

    def __init__(self, device, batch, new, equal, held, heads, kv_heads, prefix, dtype, apart=False):
        g = torch.Generator(device=device).manual_seed(batch + new)
        cpu = torch.Generator().manual_seed(3)
        self.counts = torch.full((batch,), new) if equal else torch.randint(0, new + 1, (batch,), generator=cpu)
        self.counts[-1] = new
        self.before = torch.randint(0, held + 1, (batch,), generator=cpu)
        self.n, self.P, self.equal, self.dtype, self.G, self.H = int(self.counts.sum()), prefix, equal, dtype, kv_heads, heads
        shared, width = -(-prefix // 64), -(-int((self.counts + self.before).max()) // 64)
        pages = shared + batch * width
        order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
        self.prefix, self.table = order[:shared].contiguous(), order[shared:].reshape(batch, width).contiguous()
        self.cache = paged8.Cache.empty(pages, kv_heads, device)
        for x in (self.cache.k, self.cache.v):
            x.copy_((110 * torch.randn(pages, kv_heads, 64, 128, generator=g, device=device)).clamp(-448, 448)
                    .to(torch.float8_e4m3fn))
        self.cache.scales[:, :, 0] = 120
        spread = 3 if not apart else 15 if dtype is BF16 else 7
        self.cache.scales[:, :, 1] = torch.randint(120 - spread, 121 + spread, (pages, kv_heads, 64), generator=g,
                                                   device=device).to(torch.uint8)
        self.q = torch.randn(self.n, heads, 128, generator=g, device=device).to(dtype)
        self.starts = torch.cat([torch.zeros(1, dtype=torch.long), self.counts.cumsum(0)]).to(torch.int32).to(device)
        self.lengths = (self.counts + self.before).to(torch.int32).to(device)
        self.narrow = self.n * heads // kv_heads <= 32 * batch and \
            (prefix == 0 or self.n * heads // kv_heads <= 32 or batch == 1)
        self.few = self.n * heads // kv_heads <= 32 * batch

    def run(self, bits, causal, single, **how):
        more = dict(starts=None if self.equal else self.starts, causal=causal, single_av=single, **how)
        tail = (self.prefix, self.P, self.table, self.lengths, Workspace())
        if bits == 8:
            return paged8.attention(self.q, self.cache, *tail, **more).double()
        k, v = (x.to(self.dtype).transpose(1, 2).reshape(1, -1, self.G, 128).contiguous()
                for x in oracle.pages8(self.cache))
        return paged.attention(self.q, k, v, *tail, **more).double()

    def wanted(self, causal, cap=None, slopes=None, window=None):
        """Float64 outputs, and the sums of p^2 and p^2 v^2."""
        dev, r = self.q.device, self.H // self.G
        want = torch.zeros(self.n, self.H, 128, dtype=torch.float64, device=dev)
        p2, p2v2 = torch.zeros(self.n, self.H, dtype=torch.float64, device=dev), torch.zeros_like(want)
        kp, vp = oracle.pages8(self.cache)
        lo = self.starts.tolist()
        for b, length in enumerate(self.lengths.tolist()):
            m, own, at = int(self.counts[b]), self.table[b, :-(-length // 64)].long(), slice(lo[b], lo[b + 1])
            kk, vv = (torch.cat([x[self.prefix.long()].transpose(1, 2).reshape(-1, self.G, 128)[:self.P],
                                 x[own].transpose(1, 2).reshape(-1, self.G, 128)[:length]]) for x in (kp, vp))
            place = torch.arange(len(kk), device=dev)
            mine = self.P + length - m + torch.arange(m, device=dev)[:, None]
            hidden = place > (mine if causal else self.P + length)
            if window is not None:
                hidden = hidden | (place >= self.P) & (place <= mine - window)
            for h in range(self.H):
                z = self.q[at, h].double() @ kk[:, h // r].t() * 128 ** -0.5
                if cap is not None:
                    z = cap * torch.tanh(z / cap)
                if slopes is not None:
                    z = z - slopes[h].double() * (mine - place).abs()
                p = z.masked_fill(hidden, -math.inf).softmax(-1)
                want[at, h], p2[at, h], p2v2[at, h] = p @ vv[:, h // r], (p * p).sum(-1), (p * p) @ vv[:, h // r] ** 2
        return want, p2, p2v2

    def check(self, bits, causal, **how):
        want, p2, p2v2 = self.wanted(causal, **how)
        for single in (None, False, True):
            got = self.run(bits, causal, single, **how)
            one = (not self.few if single is None else single) and not self.narrow
            # one part of the outputs' type; one of fp16 in place of two; two
            stands = bits == 8 and self.dtype is BF16 and single is not False
            parts, part = (1, None) if one else (1, FP16) if stands else (2, None)
            for h in range(self.H):
                far = float((got[:, h] - want[:, h]).norm())
                limit = float(limits.error_limit(want[:, h], p2[:, h], p2v2[:, h], self.dtype, parts, part))
                assert far <= limit, (single, h, far, limit)
            far, limit = float((got - want).norm()), float(limits.error_limit(want, p2, p2v2, self.dtype, parts, part))
            print(f'single_av={single}: {far / float(want.norm()):.3g} of the outputs, limit {limit / float(want.norm()):.3g}')
            assert far <= limit, (single, far, limit)


PLAIN = [
    # batch, new tokens, equal, held, heads, K/V heads, prefix, causal, dtype
    pytest.param(8, 1, True, 200, 8, 8, 9000, True, BF16, id='apart_narrow'),
    pytest.param(8, 1, True, 200, 8, 8, 9000, True, FP16, id='apart_narrow_fp16'),
    pytest.param(21, 1, True, 700, 6, 2, 20000, False, BF16, id='apart_two_narrow'),
    pytest.param(1, 1, True, 30, 8, 2, 30250, True, BF16, id='joint_narrow_many_pieces'),
    pytest.param(9, 1, True, 200, 3, 1, 5000, True, FP16, id='joint_narrow_pieces'),
    pytest.param(40, 3, True, 400, 12, 12, 0, True, BF16, id='joint_narrow_whole'),
    pytest.param(90, 1, True, 700, 6, 2, 20000, True, BF16, id='apart_wide_many_pieces'),
    pytest.param(64, 1, True, 600, 16, 4, 16384, True, FP16, id='apart_wide_steps'),
    pytest.param(24, 5, True, 333, 28, 4, 5003, True, BF16, id='apart_wide_more_rows'),
    pytest.param(1, 200, True, 50, 8, 2, 30000, True, BF16, id='joint_wide_many_pieces'),
    pytest.param(3, 601, True, 7, 8, 8, 126, True, FP16, id='half_wide_whole'),
    pytest.param(1, 1265, True, 134, 12, 4, 248, True, BF16, id='half_wide_causal_cut'),
    pytest.param(5, 530, False, 1600, 8, 1, 4300, False, BF16, id='ragged_prompts'),
]


@pytest.mark.parametrize('apart', [False, True], ids=['alike', 'apart'])
@pytest.mark.parametrize('batch,new,equal,held,heads,kv_heads,prefix,causal,dtype', PLAIN)
def test_rounds_as_it_says(device, batch, new, equal, held, heads, kv_heads, prefix, causal, dtype, apart):
    Call(device, batch, new, equal, held, heads, kv_heads, prefix, dtype, apart).check(8, causal)


SHAPED = [
    pytest.param(8, 1, True, 200, 8, 8, 9000, True, BF16, dict(cap=20.0, slopes=0.02), id='apart_narrow'),
    pytest.param(9, 1, True, 5000, 3, 1, 500, True, FP16, dict(window=1000), id='narrow_pieces'),
    pytest.param(40, 3, True, 400, 12, 12, 0, True, BF16, dict(slopes=0.02, window=100), id='narrow_whole'),
    pytest.param(90, 1, True, 700, 6, 2, 20000, True, BF16, dict(cap=20.0, slopes=0.02), id='apart_wide_many_pieces'),
    pytest.param(30, 7, True, 1900, 14, 2, 700, True, FP16, dict(slopes=0.02, window=300), id='wide_few_tokens'),
    pytest.param(1, 200, True, 50, 8, 2, 30000, True, BF16, dict(cap=20.0, window=64), id='wide_many_pieces'),
    pytest.param(3, 601, True, 7, 8, 8, 126, True, FP16, dict(window=200, cap=5.0), id='half_wide_whole'),
    pytest.param(1, 2000, True, 1000, 12, 12, 10, True, BF16, dict(window=900, cap=20.0), id='causal_window'),
    pytest.param(5, 530, False, 1600, 8, 1, 4300, False, BF16, dict(slopes=0.02, window=700), id='prompts'),
]


@pytest.mark.parametrize('bits', [16, 8])
@pytest.mark.parametrize('batch,new,equal,held,heads,kv_heads,prefix,causal,dtype,how', SHAPED)
def test_shaped_rounds_as_it_says(device, batch, new, equal, held, heads, kv_heads, prefix, causal, dtype, how, bits):
    how = dict(how)
    if 'slopes' in how:
        how['slopes'] = how['slopes'] * torch.exp2(-8.0 * torch.arange(heads, device=device) / heads)
    Call(device, batch, new, equal, held, heads, kv_heads, prefix, dtype).check(bits, causal, **how)
