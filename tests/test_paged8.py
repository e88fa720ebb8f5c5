"""Argument checks of the 8-bit paged cache and of shaped scores, in Python and at
the C ABI (every rejected call returns before any launch, so these run without
a GPU), the header against the binding, and the oracle against other forms."""
import ctypes
import os
import re

import pytest
import torch

from oracle import paged as plain
from oracle import paged8 as oracle
from streaming_sparse_amd import _lib, build, paged, paged8
from streaming_sparse_amd.attention import Workspace

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1
BF16 = torch.bfloat16


def args(B=2, n=3, H=4, G=2, pages=6, dtype=BF16):
    i32 = torch.int32
    return dict(q=torch.zeros(B * n, H, 128, dtype=dtype), k=torch.zeros(B * n, G, 128, dtype=dtype),
                v=torch.zeros(B * n, G, 128, dtype=dtype), cache=paged8.Cache.empty(pages, G, 'cpu'),
                table=torch.zeros(B, 2, dtype=i32), held=torch.zeros(B, dtype=i32), prefix=torch.zeros(2, dtype=i32),
                f=torch.ones(64, dtype=torch.float64))


def caches(good):
    """(error, cache) that every entry refuses."""
    k, v, s = good.k, good.v, good.scales
    pages, g = k.shape[:2]
    wide = torch.empty(pages, g, 64, 256, dtype=torch.uint8).view(torch.float8_e4m3fn)[..., :128]
    shared = k[:, :1].expand(pages, g, 64, 128)
    odd = torch.empty(k.numel() + 16, dtype=torch.uint8)[8:8 + k.numel()].view(torch.float8_e4m3fn).view(k.shape)
    return [(TypeError, paged8.Cache(k.view(torch.uint8), v, s)), (TypeError, paged8.Cache(k, v.view(torch.uint8), s)),
            (TypeError, paged8.Cache(k, v, s.float())), (TypeError, paged8.Cache(k.view(torch.float8_e5m2), v, s)),
            (ValueError, paged8.Cache(k[:1], v, s)), (ValueError, paged8.Cache(k, v, s[:1])),
            (ValueError, paged8.Cache(k[:0], v[:0], s[:0])), (ValueError, paged8.Cache(k, v, s.transpose(2, 3))),
            (ValueError, paged8.Cache(k[:, :, :32], v[:, :, :32], s)), (ValueError, paged8.Cache(wide, wide, s)),
            (ValueError, paged8.Cache(shared, shared, s)), (ValueError, paged8.Cache(odd, odd, s)),
            (ValueError, paged8.Cache(k, v.transpose(0, 1).contiguous().transpose(0, 1), s)),
            (ValueError, paged8.Cache(k, v, s[:1].expand(s.shape)))]


def test_append_rejects_bad_arguments():
    a = args()

    def bad(error=ValueError, **change):
        x = {**a, **{n: change.pop(n) for n in list(change) if n in a}}
        with pytest.raises(error):
            paged8.append(x['k'], x['v'], x['cache'], x['table'], x['held'], **{'q': x['q'], **change})

    for error, cache in caches(a['cache']):
        bad(error, cache=cache)
    bad(TypeError, k=a['k'].float())
    bad(TypeError, v=a['v'].half())
    bad(k=a['k'][..., :64])
    bad(k=a['k'][:, :1], v=a['v'][:, :1])                     # the cache's heads
    bad(q=a['q'][:5])
    bad(table=a['table'].long())
    bad(held=a['held'][:1])
    bad(starts=torch.zeros(2, dtype=torch.int32))
    bad(freqs=torch.ones(65, dtype=torch.float64))
    bad(freqs=a['f'], axes=(32, 32))                          # needs positions
    bad(freqs=a['f'], first=2 ** 53 + 1)
    bad(q=None, q_out=a['q'])
    bad(RuntimeError)                                         # none of it on a GPU


def test_read_rejects_bad_arguments():
    a = args()

    def bad(error=ValueError, cache=a['cache'], table=a['table'], first=a['held'], tokens=6, **more):
        with pytest.raises(error):
            paged8.read(cache, table, first, tokens, **more)

    for error, cache in caches(a['cache']):
        bad(error, cache=cache)
    bad(TypeError, dtype=torch.float32)
    bad(tokens=-1)
    bad(tokens=5)                                             # 2 sequences
    bad(table=a['table'].long())
    bad(table=a['table'][0])
    bad(first=a['held'][:1])
    bad(starts=torch.zeros(2, dtype=torch.int32))
    bad(k_out=a['k'][:5])
    bad(k_out=a['k'][:, :1])
    bad(TypeError, v_out=a['v'].half())
    bad(v_out=a['v'][:1].expand(6, 2, 128))                   # written rows must not overlap
    bad(RuntimeError)


def test_attention_rejects_bad_arguments():
    a = args()

    def bad(error=ValueError, prefix_tokens=100, **change):
        x = {**a, **{n: change.pop(n) for n in list(change) if n in a}}
        with pytest.raises(error):
            paged8.attention(x['q'], x['cache'], x['prefix'], prefix_tokens, x['table'], x['held'], Workspace(), **change)

    for error, cache in caches(a['cache']):
        bad(error, cache=cache)
    bad(TypeError, q=a['q'].float())
    bad(q=a['q'][:, :3])                                      # heads a multiple of the cache's
    bad(prefix_tokens=129)
    bad(prefix=None)
    bad(table=a['table'].t())
    bad(scale=0.0)
    bad(out=a['q'][:4])
    bad(single_av='two')
    bad(RuntimeError)


@pytest.mark.parametrize('eight', [False, True])
def test_shapes_that_are_refused(eight):
    a = args()

    def call(**shape):
        if eight:
            return paged8.attention(a['q'], a['cache'], None, 0, a['table'], a['held'], Workspace(), **shape)
        ck = torch.zeros(1, 64 * 6, 2, 128, dtype=BF16)
        return paged.attention(a['q'], ck, ck.clone(), None, 0, a['table'], a['held'], Workspace(), **shape)

    for shape in (dict(cap=0.0), dict(cap=-1.0), dict(cap=float('inf')), dict(cap=float('nan')), dict(cap=1e5),
                  dict(cap=1e-50), dict(window=0), dict(window=-5), dict(window=2.5), dict(window=float('inf')),
                  dict(window=float('nan')), dict(slopes=torch.ones(3)), dict(slopes=torch.ones(4).double()),
                  dict(slopes=torch.ones(4, 1)), dict(slopes=torch.ones(8)[::2])):
        with pytest.raises(ValueError):
            call(**shape)


def test_no_tokens_is_no_call():
    a = args(n=0)
    assert paged8.append(a['k'], a['v'], a['cache'], a['table'], a['held'], q=a['q']).shape == (0, 4, 128)
    k, v = paged8.read(a['cache'], a['table'], a['held'], 0)
    assert k.shape == v.shape == (0, 2, 128)
    out, lse = paged8.attention(a['q'], a['cache'], None, 0, a['table'], a['held'], Workspace(), want_lse=True, cap=3.0)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)


@pytest.fixture
def no_launch(monkeypatch):
    """Calls without their launch: what the Python side alone does."""
    launched = []
    for module in (paged, paged8):
        monkeypatch.setattr(module, '_launch', lambda name, device, dev, *given: launched.append((name, given)))
    monkeypatch.setattr(paged, '_workspace_bytes', lambda key, device: 0)
    monkeypatch.setattr(paged, '_BYTES', {})
    return launched


def test_entries_that_are_called(no_launch):
    """A call's form picks its entry, each with as many arguments as it takes (the stream aside)."""
    a = args()
    ck = torch.zeros(1, 64 * 6, 2, 128, dtype=BF16)
    slopes = torch.ones(4)
    for shape, tail in ((dict(), ''), (dict(cap=2.0), '_shaped'), (dict(slopes=slopes), '_shaped'), (dict(window=7), '_shaped')):
        paged8.attention(a['q'], a['cache'], None, 0, a['table'], a['held'], Workspace(), **shape)
        paged.attention(a['q'], ck, ck.clone(), None, 0, a['table'], a['held'], Workspace(), **shape)
        assert [x[0] for x in no_launch[-2:]] == ['ssa_paged8_attention' + tail, 'ssa_paged_attention' + tail]
    paged8.append(a['k'], a['v'], a['cache'], a['table'], a['held'])
    paged8.read(a['cache'], a['table'], a['held'], 6)
    assert [x[0] for x in no_launch[-2:]] == ['ssa_paged8_append', 'ssa_paged8_read']
    for name, given in no_launch:
        assert len(given) == len(_lib.SIGNATURES[name]) - 1, name


def test_a_window_longer_than_any_sequence_is_the_longest_there_is(no_launch):
    a = args()
    for window in (1 << 30, 1 << 40):
        paged8.attention(a['q'], a['cache'], None, 0, a['table'], a['held'], Workspace(), window=window)
        assert (1 << 30) - 1 in no_launch[-1][1]


def test_read_keeps_two_buffers_of_a_workspace(no_launch):
    a, ws = args(B=1, n=60, pages=20), Workspace()
    for n in (60, 33, 64, 1):
        k, v = paged8.read(a['cache'], a['table'][:1], a['held'][:1], n, workspace=ws)
        assert k.shape == v.shape == (n, 2, 128) and k.data_ptr() != v.data_ptr()
    assert len(ws.entries) == 4


def test_half_queries_over_bfloat16_rows_are_refused(no_launch):
    """fp16 does not hold every value of rows appended as bf16; bf16 holds all of those appended as fp16."""
    a, b = args(), args(dtype=torch.float16)

    def attend(x, cache, **more):
        paged8.attention(x['q'], cache, None, 0, x['table'], x['held'], Workspace(), **more)

    cache = a['cache']
    attend(a, cache), attend(b, cache)                        # nothing is known of its rows
    paged8.append(a['k'][:0], a['v'][:0], cache, a['table'], a['held'])
    attend(b, cache)                                          # and no row is none
    paged8.append(b['k'], b['v'], cache, b['table'], b['held'])
    attend(a, cache), attend(b, cache)
    paged8.append(a['k'], a['v'], cache, a['table'], a['held'])
    calls = len(no_launch)
    for more in (dict(), dict(cap=5.0)):
        with pytest.raises(TypeError):
            attend(b, cache, **more)
    assert len(no_launch) == calls
    attend(a, cache)
    paged8.append(b['k'], b['v'], cache, b['table'], b['held'])
    with pytest.raises(TypeError):
        attend(b, cache)


def test_sources_keep_nan_semantics():
    for source in ("paged_shaped.hip", "paged8.hip", "paged8_shaped.hip"):
        flags = build.FLAGS + build.EXTRA.get(source, [])
        assert source in build.SOURCES
        assert not {"-fno-honor-nans", "-ffinite-math-only", "-ffast-math", "-Ofast"} & set(flags), source


built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libssattn.so not built")


@built
def test_header_matches_binding():
    text = open(os.path.join(ROOT, "include", "ssattn_paged8.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = {m.group(1): len(m.group(2).split(","))
             for m in re.finditer(r"\b(?:int|long long)\s+(ssa_\w+)\s*\(([^)]*)\)\s*;", text)}
    assert set(names) == {"ssa_paged8_append", "ssa_paged8_read", "ssa_paged8_attention", "ssa_paged_attention_shaped",
                          "ssa_paged8_attention_shaped", "ssa_paged8_workspace_bytes"}
    handle = ctypes.CDLL(_lib.LIB_PATH)
    for name, count in names.items():
        assert hasattr(handle, name) and len(_lib.SIGNATURES[name]) == count, name


CACHE = dict(ck=4096, cv=4096, page=16384, head=8192, scales=4096, s_page=256, s_head=128)
BAD_CACHE = [dict(ck=None), dict(cv=None), dict(scales=None), dict(ck=4100), dict(cv=4104), dict(scales=4097),
             dict(page=16392), dict(head=-8192), dict(s_page=254), dict(s_head=-128)]


def append_call(**change):
    a = dict(q=4096, q_tok=512, q_head=128, out=4096, o_tok=512, o_head=128, k=4096, k_tok=256, k_head=128, v=4096,
             v_tok=256, v_head=128, **CACHE, table=4096, held=4096, starts=None, positions=None, freqs=4096, first=0,
             tokens=0, batch=2, heads=4, kv_heads=2, pages=6, width=2, pairs=64, axis0=64, axis1=0, axes=1, flags=2,
             stream=None)
    a.update(change)
    return _lib.lib().ssa_paged8_append(*a.values())


@built
def test_append_abi_rejects():
    assert append_call() == 0                                  # no tokens: nothing launched
    for change in (dict(tokens=-1), dict(tokens=3), dict(batch=0), dict(heads=-1), dict(kv_heads=0), dict(pages=0),
                   dict(width=0), dict(pairs=65), dict(pairs=12, axis0=12, flags=0), dict(freqs=None), dict(axes=0),
                   dict(axes=2), dict(flags=4), dict(k=None), dict(v=None), dict(table=None), dict(held=None), dict(q=None),
                   dict(out=None), dict(k=4100), dict(q_tok=-512), dict(k_head=4), dict(tokens=1 << 26),
                   dict(first=2 ** 53 + 1), *BAD_CACHE):
        assert append_call(**{'tokens': 2, **change}) == INVALID, change


def read_call(**change):
    a = dict(**CACHE, table=4096, first=4096, starts=None, k=4096, k_tok=256, k_head=128, v=4096, v_tok=256, v_head=128,
             tokens=0, batch=2, kv_heads=2, pages=6, width=2, flags=0, stream=None)
    a.update(change)
    return _lib.lib().ssa_paged8_read(*a.values())


@built
def test_read_abi_rejects():
    assert read_call() == 0
    for change in (dict(tokens=-1), dict(tokens=3), dict(batch=0), dict(kv_heads=0), dict(kv_heads=32769), dict(pages=0),
                   dict(width=0), dict(flags=2), dict(table=None), dict(first=None), dict(k=None), dict(v=None), dict(k=4104),
                   dict(v_tok=-256), dict(k_head=4), dict(tokens=1 << 26), *BAD_CACHE):
        assert read_call(**{'tokens': 2, **change}) == INVALID, change


def attention_call(eight, shaped, **change):
    where = CACHE if eight else dict(ck=4096, cv=4096, kv_tok=256, kv_head=128)
    shape = dict(cap=1.0, slopes=None, window=0) if shaped else {}
    a = dict(q=4096, q_tok=512, q_head=128, **where, prefix=4096, prefix_tokens=100, table=4096, lengths=4096, starts=None,
             out=4096, o_tok=512, o_head=128, lse=None, tokens=2, batch=2, heads=4, kv_heads=2, pages=6, width=2, scale=0.1,
             **shape, flags=2, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    name = 'ssa_paged8_attention' if eight else 'ssa_paged_attention'
    return getattr(_lib.lib(), name + ('_shaped' if shaped else ''))(*a.values())


@built
@pytest.mark.parametrize('eight,shaped', [(True, False), (False, True), (True, True)])
def test_attention_abi_rejects(eight, shaped):
    changes = [dict(tokens=0), dict(tokens=3), dict(batch=0), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(pages=0),
               dict(width=0), dict(prefix_tokens=-1), dict(prefix=None), dict(scale=0.0), dict(scale=float('nan')),
               dict(scale=float('inf')), dict(flags=4), dict(flags=3 << 3), dict(flags=-1), dict(q=None), dict(table=None),
               dict(lengths=None), dict(out=None), dict(q=4098), dict(lse=4098), dict(o_tok=-8),
               dict(tokens=1 << 30, batch=1 << 10), dict(width=1 << 26)]
    changes += BAD_CACHE if eight else [dict(ck=None), dict(cv=None), dict(kv_tok=64), dict(kv_tok=260), dict(kv_tok=1 << 24)]
    if shaped:
        changes += [dict(cap=-1.0), dict(cap=float('nan')), dict(cap=float('inf')), dict(cap=65537.0),
                    dict(cap=1e-30, scale=1e20), dict(window=-1), dict(window=1 << 30),
                    dict(slopes=4098)]
    for change in changes:
        assert attention_call(eight, shaped, **change) == INVALID, change


@built
def test_workspace_sizes_of_bad_sizes():
    size = _lib.lib().ssa_paged8_workspace_bytes
    for bad in ((3, 2, 4, 2, 0, 1, 0, 1), (2, 2, 4, 3, 0, 1, 0, 1), (0, 1, 1, 1, 0, 1, 0, 1)):
        for form in ((1, 0, 0), (0, 1, 5), (1, 1, 0)):
            assert size(*bad, *form) == -1
    assert size(2, 2, 4, 2, 0, 1, 0, 1, 1, 1, -1) == -1


@pytest.mark.parametrize('dtype', [BF16, torch.float16], ids=['bf16', 'fp16'])
def test_oracle_quantises_as_a_cast_does(dtype):
    """Scaled rows through torch's own conversion; exponents of a few rows by hand."""
    x = torch.randn(500, 128, generator=torch.Generator().manual_seed(1)) * torch.logspace(-4, 4, 500)[:, None]
    x = x.to(dtype)
    y, s = oracle.quantise(x)
    scaled = x.double() * torch.exp2((127 - s).double())[:, None]
    assert torch.equal(y, scaled.float().to(torch.float8_e4m3fn).double())
    top = scaled.abs().amax(-1)
    assert (top <= 448).all() and (top > 224).all()
    for value, want in ((448.0, 127), (449.0, 128), (224.0, 126), (1.0, 127 - 8), (1.75, 127 - 8), (1.875, 127 - 7), (0.0, 1)):
        row = torch.zeros(128, dtype=torch.float32)
        row[3] = value
        assert int(oracle.exponents(row.to(BF16 if value != 449.0 else torch.float16))) == want, value


def test_oracle_attention_is_the_plain_one():
    """Without a shape, that over 16-bit pages; a window as a mask; a cap of many times the scores changes little."""
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(1, 384, 2, 128, generator=g), torch.randn(1, 384, 2, 128, generator=g)
    q = torch.randn(7, 4, 128, generator=g)
    prefix, table = torch.tensor([0, 5]), torch.tensor([[2, 3], [1, -1]])
    lengths, starts = torch.tensor([100, 70]), torch.tensor([0, 5, 7])
    for causal in (True, False):
        want = plain.attention(q, k, v, prefix, 90, table, lengths, starts, causal)
        for cap in (None, 1e6):
            got = oracle.attention(q, oracle.pages16(k), oracle.pages16(v), prefix, 90, table, lengths, starts, causal, cap=cap)
            for a, b in zip(got, want):
                assert torch.allclose(a, b, atol=1e-9)
    one = oracle.attention(q[:1], oracle.pages16(k), oracle.pages16(v), None, 0, table[:1], torch.tensor([100]),
                           torch.tensor([0, 1]), window=1)[0]
    row = v[0, 64 * 3 + 99 - 64].double().repeat_interleave(2, 0)
    assert torch.allclose(one[0], row, atol=1e-12)
    far = oracle.attention(q[:1], oracle.pages16(k), oracle.pages16(v), None, 0, table[:1], torch.tensor([100]),
                           torch.tensor([0, 1]), slopes=torch.full((4,), 1e4))[0]
    assert torch.allclose(far[0], row, atol=1e-9)
