"""The paged K/V cache in 8 bits: appending new tokens, reading rows back, and
attention behind a shared prefix (as ``paged``, at half the memory).

A row of 128 elements of one K/V head is held as e4m3 values and one power of
two, the smallest with which the row's largest magnitude stays within 448.  A
value's error is at most 2^-4 of itself, and 2^-17 of the row's largest where
that is more.  bf16 holds every value that a row stands for, so what `read`
returns and what `attention` computes with are the same numbers.

Sequences, tables, packed rows and `starts` are those of ``paged``, whose
notes on sizes hold here too.  Nothing here computes on the CPU.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .legacy_components import HEAD_DIM
from .paged import _TYPES, _append, _attend, _FAR, _ints, _launch, _overlap, _sequences, _written

PAGE = 64
_E4M3 = torch.float8_e4m3fn
_BLOCK = PAGE * HEAD_DIM         # bytes of a page of one head


@dataclass
class Cache:
    """Pages of 64 rows: values of keys and of values, and the biased exponents of
    their rows, the keys' and then the values' (x stands for x 2^(s - 127))."""
    k: torch.Tensor          # [P, G, 64, 128] float8_e4m3fn
    v: torch.Tensor
    scales: torch.Tensor     # [P, G, 2, 64] uint8
    bf16: bool = False       # whether rows were appended as bfloat16, of which fp16 may not hold the values

    @classmethod
    def empty(cls, pages, kv_heads, device):
        """A cache whose rows hold anything until they are written."""
        k, v = (torch.empty(pages, kv_heads, PAGE, HEAD_DIM, device=device, dtype=_E4M3) for _ in range(2))
        return cls(k, v, torch.empty(pages, kv_heads, 2, PAGE, device=device, dtype=torch.uint8))

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.scales))


def _cache(cache, dev):
    """(pages, K/V heads, the entries' pointers and strides) of an 8-bit cache."""
    k, v, scales = cache.k, cache.v, cache.scales
    shape, stride, s_stride = k.shape, k.stride(), scales.stride()
    if k.dtype is not _E4M3 or v.dtype is not _E4M3 or scales.dtype is not torch.uint8:
        raise TypeError("the cache must hold float8_e4m3fn values and uint8 scales")
    if len(shape) != 4 or v.shape != shape or v.stride() != stride or shape[2] != PAGE or shape[3] != HEAD_DIM or \
            shape[0] == 0 or shape[1] == 0 or scales.shape != (shape[0], shape[1], 2, PAGE):
        raise ValueError("k and v must be [P, G, 64, 128] of equal shape and strides, scales [P, G, 2, 64]")
    pages, g, _, _ = shape
    page, head, row, unit = stride
    s_page, s_head, s_row, s_unit = s_stride
    k_ptr, v_ptr, s_ptr = k.data_ptr(), v.data_ptr(), scales.data_ptr()
    if row != HEAD_DIM or unit != 1 or s_row != PAGE or s_unit != 1 or (page | head | k_ptr | v_ptr) & 15 or \
            (s_page | s_head | s_ptr) & 3 or _overlap(pages, g, page, head, _BLOCK) or \
            _overlap(pages, g, s_page, s_head, 2 * PAGE):
        raise ValueError("a page's rows of one head must lie next to each other, at multiples of 16 bytes (their "
                         "scales of 4), and not overlap another's")
    if k.get_device() != dev or v.get_device() != dev or scales.get_device() != dev:
        raise ValueError("the cache must be on the rows' device")
    return pages, g, (k_ptr, v_ptr, page, head, s_ptr, s_page, s_head)


def append(k, v, cache, table, held, *, q=None, q_out=None, starts=None, freqs=None, axes=None, positions=None,
           first=0, interleaved=True, workspace=None):
    """``paged.append`` into an 8-bit cache: keys and values are rotated and rounded
    to their 16-bit type as there, then quantised.  Infinities and NaN are held as
    NaN and do not count for their row's power of two; fp16 elements from 63488
    on are held as 61440, bf16 ones from 1.9375 * 2^127 on as 1.875 * 2^127.
    Queries stay in 16 bits."""
    code = _TYPES.get(k.dtype)
    if code is None:
        raise TypeError("k must be bfloat16 or float16")
    if not -_FAR <= first <= _FAR:
        raise ValueError("first must lie within 2^53")
    pages, g, where = _cache(cache, k.get_device())
    q = _append("ssa_paged8_append", where, pages, g, k, v, table, held, q, q_out, starts, freqs, axes, positions,
                first, interleaved, workspace, code)
    if not code and k.shape[0]:
        cache.bf16 = True
    return q


def read(cache, table, first, tokens, *, starts=None, dtype=torch.bfloat16, k_out=None, v_out=None, workspace=None):
    """Rows of the sequences in 16 bits: (k, v) [tokens, G, 128] of `dtype`, row i of
    sequence b being the sequence's row first[b] + i (first [B] int32), packed as
    the rows of ``append`` are (so what that wrote at `held` comes back with
    first=held).

    Rows outside the table, or of pages outside the cache (-1, say), come back as
    zeros; rows from starts[B] on are left alone.  bf16 holds every value exactly;
    fp16 those of rows appended as fp16, others rounded.  k_out, v_out: where the
    rows go, of any token and head strides (a 16-bit cache's rows, say); else
    buffers owned by `workspace` that the next call, of whatever size, overwrites,
    or, without one, new tensors."""
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError("dtype must be bfloat16 or float16")
    device, dev = cache.k.device, cache.k.get_device()
    pages, g, where = _cache(cache, dev)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    batch, width, table_ptr, starts_ptr = _sequences(table, starts, tokens, dev)
    first_ptr = _ints(first, "first", (batch,), dev)
    outs, places = [], []
    for name, x in (("k_out", k_out), ("v_out", v_out)):
        if x is not None:
            n, h, tok, head, ptr = _written(x, name, dtype, dev)
            if n != tokens or h != g:
                raise ValueError(f"{name} must be [tokens, G, 128]")
        else:
            tok, head, shape = g * HEAD_DIM, HEAD_DIM, (tokens, g, HEAD_DIM)
            if workspace is None:
                x = torch.empty(shape, dtype=dtype, device=device)
                ptr = x.data_ptr()
            else:
                x, ptr, _ = workspace.rows('paged_' + name, shape, device, dtype)
        outs.append(x)
        places += (ptr, tok, head)
    if tokens:
        _launch("ssa_paged8_read", device, dev, *where, table_ptr, first_ptr, starts_ptr, *places, tokens, batch, g,
                pages, width, code)
    return outs[0], outs[1]


def attention(q, cache, prefix, prefix_tokens, table, lengths, workspace, *, starts=None, causal=True, scale=None,
              want_lse=False, out=None, single_av=None, cap=None, slopes=None, window=None):
    """``paged.attention`` over an 8-bit cache, its arguments and results those of the
    16-bit one: the same numbers as attention over the rows that `read` returns, up
    to the roundings named there.  q bf16 or fp16, of the type whose rows were
    appended: fp16 queries are refused where `append` has put bf16 rows through this
    Cache, whose values fp16 need not hold (one made over filled tensors does not
    know).  Tiles of up to 32 rows take probabilities in two parts; with bf16
    queries one fp16 part (11 bits) may stand for two, but for single_av=False.
    Sums reach 2^15 times the values' size times the rows: values from 2^90 on may
    come out infinite."""
    code = _TYPES.get(q.dtype)
    if code is None:
        raise TypeError("q must be bfloat16 or float16")
    if code and cache.bf16:
        raise TypeError("float16 queries over rows that were appended as bfloat16")
    pages, g, where = _cache(cache, q.get_device())
    return _attend("ssa_paged8_attention", True, where, pages, g, q, prefix, prefix_tokens, table, lengths, workspace,
                   starts, causal, scale, want_lse, out, single_av, cap, slopes, window, code)
