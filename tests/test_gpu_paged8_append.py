"""What an append into the 8-bit cache writes, bit for bit."""
import pytest
import torch

from oracle import paged as plain
from oracle import paged8 as oracle
from streaming_sparse_amd import paged8

BF16, FP16 = torch.bfloat16, torch.float16


def one_sequence(device, k, v, dtype, **more):
    """Rows k, v [N, G, 128] appended to an empty cache: (cache, k and v read back)."""
    n, g = k.shape[:2]
    width = -(-n // 64)
    cache = paged8.Cache.empty(width, g, device)
    table = torch.arange(width, dtype=torch.int32, device=device)[None]
    held = torch.zeros(1, dtype=torch.int32, device=device)
    paged8.append(k, v, cache, table, held, **more)
    return (cache, *paged8.read(cache, table, held, n, dtype=dtype))


def ends(dtype):
    """Rows that hold the 256 largest values of a type, of either sign, in rows of every size of others."""
    top = 0x7bff if dtype is FP16 else 0x7f7f
    x = torch.arange(top - 255, top + 1).to(torch.int16).view(dtype)
    x = torch.cat([x, -x])
    rows = torch.zeros(512, 1, 128, dtype=dtype)
    for i in range(512):
        rows[i, 0, i % 128] = x[i]
        rows[i, 0, 5:70] = torch.where(rows[i, 0, 5:70] == 0, x.flip(0)[i // 2] * 2.0 ** -(i % 11), rows[i, 0, 5:70])
    return rows


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
def test_oracle_keeps_the_largest_values_finite(dtype):
    x = ends(dtype)
    y = oracle.values(*oracle.quantise(x))
    assert (y.abs() <= torch.finfo(dtype).max).all()
    # off by half a step, an eighth of the values' power of two, or by as much as the last value is cut
    assert ((y - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -17 * x.double().abs().amax(-1, keepdim=True)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
def test_finite_values_stay_finite(device, dtype):
    """The ends of the type, and all its finite values, come back finite in their own type and as the oracle has them."""
    every = torch.arange(-32768, 32768).to(torch.int16).view(dtype)
    every = torch.where(torch.isfinite(every.double()), every, torch.zeros_like(every)).reshape(-1, 1, 128)
    x = torch.cat([ends(dtype), every]).to(device)
    cache, k, v = one_sequence(device, x, x.flip(0), dtype)
    for got, given in ((k, x), (v, x.flip(0))):
        assert torch.isfinite(got).all()
        want, s = oracle.quantise(given)
        # fp16 rounds those below its smallest normal value
        assert torch.equal(got, oracle.values(want, s).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('interleaved', [True, False], ids=['pairs', 'halves'])
@pytest.mark.parametrize('dtype', [BF16, FP16], ids=['bf16', 'fp16'])
def test_keys_turn_in_float64(device, dtype, interleaved):
    """16 million elements of turned keys as float64 has them, rounded to float32, to 16 bits and to 8: bit for bit.
    Angles of up to 8192 radians are off by 2^-40, which brings an element to another 16-bit value with a chance of
    2^-40 / 2^-12 at most; a turn in float32 does so to an 8-bit value of every 10^5, leaving out the rounding to
    float32 to one of every 2 x 10^6."""
    n, g = 8192, 16
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn(n, g, 128, generator=gen).to(dtype) for _ in range(2))
    freqs = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    turned = plain.rotate(k.double(), torch.arange(n)[:, None], freqs, (64,), interleaved).float().to(dtype)
    cache, got_k, got_v = one_sequence(device, k.to(device), v.to(device), dtype, freqs=freqs.to(device),
                                       interleaved=interleaved)
    for got, given in ((got_k, turned), (got_v, v)):
        want, s = oracle.quantise(given.to(device))
        want = oracle.values(want, s).to(dtype)
        off = int((got != want).sum())
        assert off == 0, off
