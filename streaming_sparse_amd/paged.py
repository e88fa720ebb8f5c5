"""Several sequences over one paged K/V cache: appending new tokens with their
position rotation, and attention of all of them behind a shared prefix.

The cache is the resident one of the attention path, [1, 64 P, G, 128] for G
K/V heads (token-major, or head-major strided); a page is 64 of its rows.  A
sequence (a continuation of one history, a candidate of one step) owns pages
through a row of ``table`` [B, M] int32; a list ``prefix`` of pages lies
before every sequence.  The new tokens of all sequences are packed, sequence
b's at rows starts[b] .. starts[b + 1] - 1 of [N, heads, 128] tensors (starts
None: N / B each).

Every size on the host is a bound only: how many tokens a sequence holds and
where its rows start are read on the device, so a captured call is replayed
with other values.  Nothing here computes on the CPU.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .legacy_components import HEAD_DIM, kv_strides

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_INT, _F64 = torch.int32, torch.float64
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, '_cuda_getDevice') else torch.cuda.current_device


def _cache(cache_k, cache_v, dtype, device):
    """(pages, K/V heads, token stride, head stride) of the resident cache."""
    shape = cache_k.shape
    if len(shape) != 4 or shape[0] != 1 or shape[3] != HEAD_DIM or shape[1] == 0 or shape[1] % 64 or \
            cache_v.shape != shape:
        raise ValueError("cache_k and cache_v must be [1, 64P, G, 128] of equal shape")
    if cache_k.dtype is not dtype or cache_v.dtype is not dtype:
        raise TypeError("the cache must have the new rows' dtype (bfloat16 or float16)")
    if cache_k.device != device or cache_v.device != device:
        raise ValueError("the cache must be on the new rows' device")
    tok, head = kv_strides(cache_k, cache_v)
    return shape[1] // 64, shape[2], tok, head


def _rows(x, name, dtype, device):
    """(token stride, head stride) of packed rows [N, heads, 128]."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1:
        raise ValueError(f"{name} must be [N, heads, 128] with adjacent elements in a row")
    if x.dtype is not dtype or x.device != device:
        raise TypeError(f"{name} must share the other rows' dtype and device")
    if (stride[0] | stride[1]) & 7 or x.data_ptr() & 15:
        raise ValueError(f"{name}'s rows must start at multiples of 16 bytes")
    return stride[0], stride[1]


def _ints(x, name, shape, device):
    if x.dtype is not _INT or x.shape != shape or not x.is_contiguous() or x.device != device:
        raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the rows' device")
    return x.data_ptr()


def _sequences(table, starts, tokens, device):
    """(batch, pages a sequence may own, starts pointer)."""
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError("table must be [B, M]")
    batch, width = table.shape
    if starts is None:
        if tokens % batch:
            raise ValueError("without starts, the sequences have N / B new tokens each: N must be a multiple of B")
        return batch, width, None
    return batch, width, _ints(starts, "starts", (batch + 1,), device)


def _on(device, call):
    """call() with `device` current."""
    if device.type != 'cuda':
        raise RuntimeError("the tensors must be on a GPU")
    if device.index is None or device.index == _current_device():
        return call()
    with torch.cuda.device(device):
        return call()


def append(k, v, cache_k, cache_v, table, held, *, q=None, q_out=None, starts=None, freqs=None, axes=None,
           positions=None, first=0, interleaved=True, workspace=None):
    """Keys and values of the sequences' new tokens into the cache, keys and
    queries rotated on the way; returns the rotated queries (None without q).

    k, v [N, G, 128], q [N, H, 128]: bf16 or fp16 rows, of any token and head
    strides (parts of one projection's output, say).  Token i of sequence b
    becomes the sequence's row held[b] + i (held [B] int32: the tokens it has
    already).  Tokens whose row lies outside the table or whose page outside
    the cache (-1, say) are not written; rows from starts[B] on are left
    alone.  Two tokens of a call must not share a cache row.

    freqs [R] float64: radians per position of the first R pairs (R <= 64;
    None: no rotation), elements (2j, 2j+1) with `interleaved`, else (j, j+R)
    with R a multiple of 8.  A token's position is first + held[b] + i, or
    given by `positions` int32 [N] or [N, A]: the first axes[0] pairs turn on
    the first axis, and so on (axes: up to 3 counts that sum to R).  Angles
    are formed in float64.

    q_out: where the rotated queries go (q itself is allowed); else a buffer
    owned by `workspace` that the next call overwrites, or, without one, a new
    tensor."""
    device, dtype = k.device, k.dtype
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError("k must be bfloat16 or float16")
    k_tok, k_head = _rows(k, "k", dtype, device)
    v_tok, v_head = _rows(v, "v", dtype, device)
    n, g, _ = k.shape
    pages, gc, kv_tok, kv_head = _cache(cache_k, cache_v, dtype, device)
    if v.shape != k.shape or gc != g:
        raise ValueError("k and v must be [N, G, 128] for the cache's G heads")
    batch, width, starts_ptr = _sequences(table, starts, n, device)
    table_ptr, held_ptr = _ints(table, "table", (batch, width), device), _ints(held, "held", (batch,), device)
    pairs, a0, a1, na, freqs_ptr, pos_ptr = 0, 0, 0, 1, None, None
    if freqs is not None:
        if freqs.dtype is not _F64 or freqs.dim() != 1 or freqs.device != device or not freqs.is_contiguous():
            raise ValueError("freqs must be a contiguous float64 [R] tensor on the rows' device")
        pairs, freqs_ptr = freqs.shape[0], freqs.data_ptr()
        if pairs > HEAD_DIM // 2 or (not interleaved and pairs % 8):
            raise ValueError("at most 64 pairs, a multiple of 8 in halves")
        counts = (pairs,) if axes is None else tuple(axes)
        na = len(counts)
        if not 1 <= na <= 3 or sum(counts) != pairs or min(counts) < 0:
            raise ValueError("axes must be 1 to 3 counts that sum to the pairs")
        a0, a1 = counts[0], counts[1] if na > 1 else 0
        if positions is not None:
            pos_ptr = _ints(positions, "positions", (n,) if positions.dim() == 1 and na == 1 else (n, na), device)
        elif na > 1:
            raise ValueError("several axes need positions")
    elif positions is not None or axes is not None:
        raise ValueError("positions and axes need freqs")
    h, q_ptr, out_ptr, q_tok, q_head, o_tok, o_head = 0, None, None, 0, 0, 0, 0
    if q is not None:
        q_tok, q_head = _rows(q, "q", dtype, device)
        h = q.shape[1]
        if q.shape[0] != n or h == 0:
            raise ValueError("q must be [N, H, 128]")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=device) if workspace is None else \
                workspace.tensor('paged_q', q.shape, device, dtype)
        elif q_out.shape != q.shape:
            raise ValueError("q_out must have q's shape")
        o_tok, o_head = _rows(q_out, "q_out", dtype, device)
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    if n == 0:
        return q_out
    _on(device, lambda: _lib.check(_lib.lib().ssa_paged_append(
        q_ptr, q_tok, q_head, out_ptr, o_tok, o_head, k.data_ptr(), k_tok, k_head, v.data_ptr(), v_tok, v_head,
        cache_k.data_ptr(), cache_v.data_ptr(), kv_tok, kv_head, table_ptr, held_ptr, starts_ptr, pos_ptr, freqs_ptr,
        first, n, batch, h, g, pages, width, pairs, a0, a1, na, code | (2 if interleaved else 0),
        _lib.stream_handle(device)), "ssa_paged_append"))
    return q_out


_BYTES = {}


def attention(q, cache_k, cache_v, prefix, prefix_tokens, table, lengths, workspace, *, starts=None, causal=True,
              scale=None, want_lse=False, out=None):
    """Attention of every sequence's new queries over the shared prefix and the
    sequence's own rows; the prefix is read for all sequences together.

    q [N, H, 128] bf16 or fp16, any token and head strides; H a multiple of
    the cache's G heads, query head h on K/V head h // (H / G).  prefix int32
    [>= ceil(prefix_tokens / 64)]: the shared pages, all sequences see their
    first prefix_tokens rows (prefix may be None with prefix_tokens 0).
    lengths [B] int32: rows of each sequence in the cache, the new tokens'
    among them.  Query i of n attends the prefix and its sequence's rows j <
    lengths[b], with `causal` only j <= lengths[b] - n + i.  A query that
    sees nothing gets zeros (and lse -inf).  Rows from starts[B] on are left
    as they were.  Pages outside the cache (-1) count as absent; rows that no
    query sees may hold anything, while a value row that some query of the
    call sees must be finite for the others to come out finite.

    scale defaults to 128 ** -0.5.  Returns out [N, H, 128], or (out, lse)
    with want_lse, lse [N, H] float32 the log of the sum of exponentials:
    buffers owned by `workspace` and overwritten by the next call, or `out` as
    given.

    Arithmetic: scores, maxima, sums and the joins of pieces are float32.  A
    probability meets V in 16 bits: in two parts (hi + lo) where a tile is
    bound by memory, in one where by the matrix pipe (fp16: scaled up by
    2^7)."""
    device, dtype = q.device, q.dtype
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError("q must be bfloat16 or float16")
    q_tok, q_head = _rows(q, "q", dtype, device)
    n, h, _ = q.shape
    pages, g, kv_tok, kv_head = _cache(cache_k, cache_v, dtype, device)
    if h == 0 or h % g:
        raise ValueError("the query heads must be a multiple of the cache's heads")
    batch, width, starts_ptr = _sequences(table, starts, n, device)
    table_ptr, len_ptr = _ints(table, "table", (batch, width), device), _ints(lengths, "lengths", (batch,), device)
    prefix_ptr = None
    if prefix_tokens < 0:
        raise ValueError("prefix_tokens must not be negative")
    if prefix_tokens > 0:
        if prefix is None or prefix.dim() != 1 or 64 * prefix.shape[0] < prefix_tokens:
            raise ValueError("prefix must list the pages of prefix_tokens rows")
        prefix_ptr = _ints(prefix, "prefix", prefix.shape, device)
    scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive")
    if out is None:
        out = workspace.tensor('paged_out', q.shape, device, dtype)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape")
    o_tok, o_head = _rows(out, "out", dtype, device)
    lse = workspace.tensor('paged_lse', (n, h), device, torch.float32) if want_lse else None
    if n:
        _on(device, lambda: _attend(
            q.data_ptr(), q_tok, q_head, cache_k.data_ptr(), cache_v.data_ptr(), kv_tok, kv_head, prefix_ptr,
            prefix_tokens, table_ptr, len_ptr, starts_ptr, out.data_ptr(), o_tok, o_head,
            None if lse is None else lse.data_ptr(), n, batch, h, g, pages, width, scale,
            code | (2 if causal else 0), workspace, device))
    return (out, lse) if want_lse else out


def _attend(*args):
    *call, workspace, device = args
    starts, prefix_tokens = call[11], call[8]
    tokens, batch, heads, kv_heads, _, width = call[16:22]
    key = (tokens, batch, heads, kv_heads, prefix_tokens, width, starts is not None, device)
    need = _BYTES.get(key)
    if need is None:
        need = _lib.lib().ssa_paged_attention_workspace_bytes(tokens, batch, heads, kv_heads, prefix_tokens, width,
                                                              int(starts is not None))
        if need < 0:
            raise ValueError("paged.attention: sizes out of range")
        if len(_BYTES) > 4096:
            _BYTES.clear()
        _BYTES[key] = need
    part = workspace.tensor('paged_part', (need,), device, torch.uint8).data_ptr() if need else None
    _lib.check(_lib.lib().ssa_paged_attention(*call, part, need, _lib.stream_handle(device)), "ssa_paged_attention")
