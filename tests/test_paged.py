"""Argument checks of the paged append and the shared-prefix attention, in
Python and at the C ABI (every rejected call returns before any launch, so
these run without a GPU), the header against the binding, and the oracle
against whole-sequence formulas."""
import ctypes
import os
import re

import pytest
import torch

from oracle import paged as oracle
from streaming_sparse_amd import _lib, build, paged
from streaming_sparse_amd.attention import Workspace

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1


def args(B=2, n=3, H=4, G=2, pages=6, dtype=torch.bfloat16):
    i32 = torch.int32
    return dict(q=torch.zeros(B * n, H, 128, dtype=dtype), k=torch.zeros(B * n, G, 128, dtype=dtype),
                v=torch.zeros(B * n, G, 128, dtype=dtype), ck=torch.zeros(1, 64 * pages, G, 128, dtype=dtype),
                cv=torch.zeros(1, 64 * pages, G, 128, dtype=dtype), table=torch.zeros(B, 2, dtype=i32),
                held=torch.zeros(B, dtype=i32), prefix=torch.zeros(2, dtype=i32),
                f=torch.ones(64, dtype=torch.float64))


def test_append_rejects_bad_arguments():
    a = args()

    def bad(error=ValueError, **change):
        x = {**a, **{n: change.pop(n) for n in list(change) if n in a}}
        with pytest.raises(error):
            paged.append(x['k'], x['v'], x['ck'], x['cv'], x['table'], x['held'], **{'q': x['q'], **change})

    bad(TypeError, k=a['k'].float())
    bad(TypeError, v=a['v'].half())
    bad(TypeError, ck=a['ck'].half(), cv=a['cv'].half())
    bad(k=a['k'][..., :64])
    bad(v=a['v'][:4])
    bad(k=a['k'][:, :1], v=a['v'][:, :1])                     # the cache's heads
    bad(ck=a['ck'][:, :100], cv=a['cv'][:, :100])             # whole pages
    bad(cv=a['cv'][:, :64])
    bad(k=torch.zeros(6, 2, 256, dtype=torch.bfloat16)[..., ::2])
    bad(k=torch.zeros(6, 2, 132, dtype=torch.bfloat16)[..., :128])      # rows at 16 bytes
    bad(q=a['q'][:5])
    bad(table=a['table'].long())
    bad(table=a['table'][0])
    bad(held=a['held'][:1])
    bad(starts=torch.zeros(2, dtype=torch.int32))
    bad(table=torch.zeros(4, 2, dtype=torch.int32), held=torch.zeros(4, dtype=torch.int32))    # 6 tokens, 4 sequences
    bad(freqs=a['f'].float())
    bad(freqs=torch.ones(65, dtype=torch.float64))
    bad(freqs=torch.ones(12, dtype=torch.float64), interleaved=False)
    bad(freqs=a['f'], axes=(30, 30))
    bad(freqs=a['f'], axes=(16, 16, 16, 16))
    bad(freqs=a['f'], axes=(32, 32))                          # needs positions
    bad(freqs=a['f'], axes=(70, -6), positions=torch.zeros(6, 2, dtype=torch.int32))
    bad(freqs=a['f'], axes=(32, 32), positions=torch.zeros(6, 3, dtype=torch.int32))
    bad(freqs=a['f'], positions=torch.zeros(6, dtype=torch.int64))
    bad(positions=torch.zeros(6, dtype=torch.int32))
    bad(q_out=a['q'][:5])
    bad(q_out=a['q'][:, :1].expand(6, 4, 128))               # written rows must not overlap
    bad(q=None, q_out=a['q'])
    bad(ck=a['ck'][:, :, :1].expand(1, 384, 2, 128), cv=a['cv'][:, :, :1].expand(1, 384, 2, 128))
    bad(cv=torch.zeros(1, 2, 384, 128, dtype=torch.bfloat16).transpose(1, 2))     # k and v in one layout


def test_attention_rejects_bad_arguments():
    a = args()

    def bad(error=ValueError, prefix_tokens=100, **change):
        x = {**a, **{n: change.pop(n) for n in list(change) if n in a}}
        with pytest.raises(error):
            paged.attention(x['q'], x['ck'], x['cv'], x['prefix'], prefix_tokens, x['table'], x['held'], Workspace(),
                            **change)

    bad(TypeError, q=a['q'].float())
    bad(TypeError, q=a['q'].half())
    bad(q=a['q'][:, :3])                                      # heads a multiple of the cache's
    bad(q=a['q'][..., :64])
    bad(prefix_tokens=129)
    bad(prefix_tokens=-1)
    bad(prefix=None)
    bad(prefix=a['prefix'].long())
    bad(table=a['table'].t())
    bad(held=a['held'].long())
    bad(starts=torch.zeros(3, dtype=torch.int64))
    bad(scale=0.0)
    bad(scale=float('nan'))
    bad(out=a['q'][:4])
    bad(out=a['q'][:1].expand(6, 4, 128))
    bad(TypeError, out=a['q'].half())
    bad(table=torch.zeros(5, 2, dtype=torch.int32), held=torch.zeros(5, dtype=torch.int32))


def test_no_tokens_is_no_call():
    """Zero new tokens launch nothing (no library call is made, so this runs without a GPU)."""
    a = args(n=0)
    assert paged.append(a['k'], a['v'], a['ck'], a['cv'], a['table'], a['held'], q=a['q']).shape == (0, 4, 128)
    out, lse = paged.attention(a['q'], a['ck'], a['cv'], None, 0, a['table'], a['held'], Workspace(), want_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)


def test_paged_sources_keep_nan_semantics():
    """Rows that no query sees may hold NaN, and a NaN that is seen reaches the
    output: neither source may be compiled as if there were none."""
    for source in ("paged.hip", "append.hip"):
        flags = build.FLAGS + build.EXTRA.get(source, [])
        assert source in build.SOURCES
        assert not {"-fno-honor-nans", "-ffinite-math-only", "-ffast-math", "-Ofast"} & set(flags), source


@pytest.fixture
def no_launch(monkeypatch):
    """Calls without their launch: what the Python side alone does."""
    launched = []
    monkeypatch.setattr(paged, '_launch', lambda name, device, dev, *given: launched.append((name, given)))
    monkeypatch.setattr(paged, '_workspace_bytes', lambda key, device: 0)
    monkeypatch.setattr(paged, '_BYTES', {})
    return launched


def test_calls_of_many_sizes_share_a_few_buffers(no_launch):
    """A workspace that sees every token count up to 600 keeps one buffer per power
    of two for queries, outputs and lse, less than four times the largest together."""
    a, ws = args(B=1, n=600, pages=20), Workspace()
    for n in (*range(1, 601), 37, 600, 1):
        q, k, v = a['q'][:n], a['k'][:n], a['v'][:n]
        turned = paged.append(k, v, a['ck'], a['cv'], a['table'], a['held'], q=q, workspace=ws)
        out, lse = paged.attention(turned, a['ck'], a['cv'], None, 0, a['table'], a['held'], ws, want_lse=True)
        assert turned.shape == out.shape == q.shape and lse.shape == q.shape[:2]
        assert turned.is_contiguous() and out.is_contiguous() and lse.is_contiguous()
        assert turned.data_ptr() != out.data_ptr()
    assert len(no_launch) == 2 * 603 and len(ws.entries) == 3 * 11
    assert ws.bytes() < 4 * 600 * 4 * (2 * 256 + 4)


def test_rows_in_the_buffer_that_is_written(no_launch):
    """A result that lies in the workspace may come back as it stands, whatever the
    next call's size; other parts of its buffer are refused."""
    a, ws = args(B=1, n=12, H=2, pages=20), Workspace()
    turn = lambda q, k, v: paged.append(k, v, a['ck'], a['cv'], a['table'], a['held'], q=q, workspace=ws)
    see = lambda q: paged.attention(q, a['ck'], a['cv'], None, 0, a['table'], a['held'], ws)
    q = turn(a['q'], a['k'], a['v'])
    assert turn(q, a['k'], a['v']).data_ptr() == q.data_ptr()
    assert turn(q[:9], a['k'][:9], a['v'][:9]).data_ptr() == q.data_ptr()
    for bad in (q[1:10], q.as_strided((9, 2, 128), (128, 128, 1)), q[:9, 1:].expand(9, 2, 128)):
        with pytest.raises(ValueError):
            turn(bad, a['k'][:9], a['v'][:9])
    for part in (q[:9], q[3:12]):
        with pytest.raises(ValueError):
            turn(a['q'][:9], part, a['v'][:9])
        with pytest.raises(ValueError):
            turn(a['q'][:9], a['k'][:9], part)
    out = see(q)
    assert see(out).data_ptr() == see(out[:9]).data_ptr() == out.data_ptr()
    for bad in (out[1:10], out.as_strided((9, 2, 128), (128, 128, 1)), out[:9, 1:].expand(9, 2, 128)):
        with pytest.raises(ValueError):
            see(bad)
    one = args(B=1, n=1, H=1, G=1, pages=2)
    q = paged.append(one['k'], one['v'], one['ck'], one['cv'], one['table'], one['held'], q=one['q'], workspace=ws)
    with pytest.raises(ValueError):
        paged.append(q, one['v'], one['ck'], one['cv'], one['table'], one['held'], q=one['q'], workspace=ws)


built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libssattn.so not built")


def declared():
    text = open(os.path.join(ROOT, "include", "ssattn_paged.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return {m.group(1): len(m.group(2).split(","))
            for m in re.finditer(r"\b(?:int|long long)\s+(ssa_\w+)\s*\(([^)]*)\)\s*;", text)}


@built
def test_header_matches_binding():
    names = declared()
    assert set(names) == {"ssa_paged_append", "ssa_paged_attention", "ssa_paged_attention_workspace_bytes"}
    handle = ctypes.CDLL(_lib.LIB_PATH)
    for name, count in names.items():
        assert hasattr(handle, name) and len(_lib.SIGNATURES[name]) == count, name


def append_call(**change):
    a = dict(q=4096, q_tok=512, q_head=128, out=4096, o_tok=512, o_head=128, k=4096, k_tok=256, k_head=128, v=4096,
             v_tok=256, v_head=128, ck=4096, cv=4096, kv_tok=256, kv_head=128, table=4096, held=4096, starts=None,
             positions=None, freqs=4096, first=0, tokens=0, batch=2, heads=4, kv_heads=2, pages=6, width=2, pairs=64,
             axis0=64, axis1=0, axes=1, flags=2, stream=None)
    a.update(change)
    return _lib.lib().ssa_paged_append(*a.values())


@built
def test_append_abi_rejects():
    assert append_call() == 0                                  # no tokens: nothing launched
    for change in (dict(tokens=-1), dict(tokens=3), dict(batch=0), dict(heads=-1), dict(kv_heads=0), dict(pages=0),
                   dict(width=0), dict(pairs=65), dict(pairs=-1), dict(pairs=12, axis0=12, flags=0), dict(freqs=None),
                   dict(axes=0), dict(axes=4), dict(axis0=65), dict(axis0=40, axis1=40), dict(axes=2), dict(flags=4),
                   dict(k=None), dict(v=None), dict(ck=None), dict(cv=None), dict(table=None), dict(held=None),
                   dict(q=None), dict(out=None), dict(k=4100), dict(kv_tok=260), dict(q_tok=-512), dict(k_head=4),
                   dict(kv_tok=64), dict(tokens=1 << 26)):
        assert append_call(**{'tokens': 2, **change}) == INVALID, change


@built
def test_append_abi_rejects_pairs_beyond_the_axes():
    """Positions hold `axes` numbers a token: no pair may turn on one behind them,
    which for the last token would lie outside the tensor."""
    for change in (dict(axis0=63), dict(axis0=0), dict(axis0=32, axis1=32), dict(axis0=40, axis1=20),
                   dict(axes=2, axis0=32, axis1=31), dict(axes=2, axis0=0, axis1=0), dict(axes=2, axis0=63)):
        assert append_call(**{'tokens': 2, 'positions': 4096, **change}) == INVALID, change
    for change in (dict(), dict(axes=2, axis0=32, axis1=32), dict(axes=2, axis0=64), dict(axes=3, axis0=22, axis1=21),
                   dict(axes=3, axis0=0)):
        assert append_call(**{'positions': 4096, **change}) == 0, change


@built
@pytest.mark.parametrize('tokens', [(1 << 26) - 3, (1 << 26) - 2, (1 << 26) - 1])
def test_append_abi_rejects_tokens_that_no_grid_holds(tokens):
    """2^24 workgroups of 256 threads are 2^32 threads."""
    assert append_call(tokens=tokens, batch=1) == INVALID


def attention_call(**change):
    a = dict(q=4096, q_tok=512, q_head=128, ck=4096, cv=4096, kv_tok=256, kv_head=128, prefix=4096, prefix_tokens=100,
             table=4096, lengths=4096, starts=None, out=4096, o_tok=512, o_head=128, lse=None, tokens=2, batch=2,
             heads=4, kv_heads=2, pages=6, width=2, scale=0.1, flags=2, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return _lib.lib().ssa_paged_attention(*a.values())


@built
def test_attention_abi_rejects():
    for change in (dict(tokens=0), dict(tokens=3), dict(batch=0), dict(heads=3), dict(heads=0), dict(kv_heads=0),
                   dict(pages=0), dict(width=0), dict(prefix_tokens=-1), dict(prefix=None), dict(scale=0.0),
                   dict(scale=float('nan')), dict(scale=float('inf')), dict(flags=4), dict(q=None), dict(ck=None),
                   dict(cv=None), dict(table=None), dict(lengths=None), dict(out=None), dict(q=4098), dict(lse=4098),
                   dict(kv_tok=64), dict(kv_tok=260), dict(o_tok=-8), dict(tokens=1 << 30, batch=1 << 10), dict(width=1 << 26), dict(kv_tok=1 << 24)):
        assert attention_call(**change) == INVALID, change
    size = _lib.lib().ssa_paged_attention_workspace_bytes
    assert size(3, 2, 4, 2, 0, 1, 0, 1) == -1 and size(2, 2, 4, 3, 0, 1, 0, 1) == -1 and size(0, 1, 1, 1, 0, 1, 0, 1) == -1


def test_oracle_attention_is_dense_attention():
    """One sequence, pages in order: the oracle equals softmax(q k^T) v over prefix
    and own rows, causal and not."""
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(1, 256, 2, 128, generator=g), torch.randn(1, 256, 2, 128, generator=g)
    q = torch.randn(5, 4, 128, generator=g)
    prefix, table = torch.tensor([0, 1]), torch.tensor([[2, 3]])
    for causal in (True, False):
        out, lse, _ = oracle.attention(q, k, v, prefix, 128, table, torch.tensor([100]), torch.tensor([0, 5]), causal)
        kk, vv = (x[0, :228].double().repeat_interleave(2, 1) for x in (k, v))
        z = torch.einsum('qhd,khd->hqk', q.double(), kk) / 128 ** 0.5
        if causal:
            z = z.masked_fill(torch.arange(228) > 223 + torch.arange(5)[:, None], float('-inf'))
        want = torch.einsum('hqk,khd->qhd', z.softmax(-1), vv)
        assert torch.allclose(out, want, atol=1e-12) and torch.allclose(lse, z.logsumexp(-1).t(), atol=1e-12)


def test_oracle_rotation_is_complex_multiplication():
    g = torch.Generator().manual_seed(5)
    x, f = torch.randn(3, 2, 128, generator=g, dtype=torch.float64), torch.rand(64, generator=g, dtype=torch.float64)
    pos = torch.tensor([[0], [5], [-11]])
    z = torch.polar(torch.ones(3, 64, dtype=torch.float64), pos * f)[:, None]
    w = torch.view_as_real(torch.view_as_complex(x.reshape(3, 2, 64, 2)) * z).reshape(3, 2, 128)
    assert torch.allclose(oracle.rotate(x, pos, f, (64,), True), w, atol=1e-12)
    halves = torch.cat([x[..., 0::2], x[..., 1::2]], -1)
    want = torch.cat([w[..., 0::2], w[..., 1::2]], -1)
    assert torch.allclose(oracle.rotate(halves, pos, f, (64,), False), want, atol=1e-12)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('keys', [300, 2000, 30250])
def test_error_limit_tells_wrong_outputs(keys, dtype):
    """The limit holds for outputs rounded once, with probabilities in two parts or
    one, and is passed by far by mistakes planted in the float64 form: a page
    of V left out, two half pages exchanged, and, against the limit of two
    parts over a few thousand outputs, probabilities in one part."""
    g = torch.Generator().manual_seed(keys)
    rows = 16
    q, k, v = (torch.randn(n, 128, generator=g).to(dtype).double() for n in (rows, keys, keys))
    p = (q @ k.t() * 128 ** -0.5).softmax(-1)
    want, p2, p2v2 = p @ v, (p * p).sum(-1), (p * p) @ (v * v)

    # as a tile forms them: beside the row's largest, in fp16 2^7 times as large
    unit = p.amax(-1, keepdim=True) / (128 if dtype is torch.float16 else 1)

    def part(x):
        return (x / unit).to(dtype).double() * unit

    def size(out, rows=slice(None)):
        return (out.to(dtype).double() - want)[rows].norm()

    def limit(parts, r=slice(None)):
        return oracle.error_limit(want[r], p2[r], p2v2[r], dtype, parts)

    hi = part(p)
    both = hi + part(p - hi)
    assert size(both @ v) <= limit(2) and size(hi @ v) <= limit(1)
    assert size(hi @ v) > limit(2)
    for r in range(rows):
        assert size(both @ v, [r]) <= limit(2, [r]) and size(hi @ v, [r]) <= limit(1, [r])
    at = keys // 128 * 64
    lost, moved = v.clone(), v.clone()
    lost[at:at + 64] = 0
    moved[at:at + 32], moved[at + 32:at + 64] = v[at + 32:at + 64], v[at:at + 32]
    for bad in (lost, moved):
        for r in range(rows):
            assert size(p @ bad, [r]) > 3 * limit(1, [r])


def test_attention_rejects_what_is_no_precision():
    a = args()
    for value in ('two', 2, 0.5):
        with pytest.raises(ValueError):
            paged.attention(a['q'], a['ck'], a['cv'], a['prefix'], 100, a['table'], a['held'], Workspace(),
                            single_av=value)


@built
def test_attention_abi_rejects_unknown_flags():
    for flags in (3 << 3, 1 << 5, 4 | 1 << 3, -1):
        assert attention_call(flags=flags) == INVALID, flags


@built
def test_append_rejects_a_first_position_that_float64_cannot_count(no_launch):
    """Positions are counted in 64 bits and become float64: `first` beyond 2^53 would
    be taken for another, or wrap."""
    a = args()
    for first in (2 ** 53 + 1, -2 ** 53 - 1, 2 ** 63, 2 ** 64 + 5):
        with pytest.raises(ValueError):
            paged.append(a['k'], a['v'], a['ck'], a['cv'], a['table'], a['held'], freqs=a['f'], first=first)
    for first in (2 ** 53, -2 ** 53, 0):
        paged.append(a['k'], a['v'], a['ck'], a['cv'], a['table'], a['held'], freqs=a['f'], first=first)
    assert [given[21] for _, given in no_launch] == [2 ** 53, -2 ** 53, 0]
    for first in (2 ** 53 + 1, -2 ** 53 - 1, 2 ** 63 - 1, -2 ** 63):
        assert append_call(first=first) == INVALID
    assert append_call(first=2 ** 53) == append_call(first=-2 ** 53) == 0
