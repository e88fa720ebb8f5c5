"""Several sequences over one paged K/V cache: appending new tokens with their
position rotation, and attention of all of them behind a shared prefix.

The cache is the resident one of the attention path, [1, 64 P, G, 128] for G
K/V heads (token-major, or head-major strided); a page is 64 of its rows.  A
sequence (a continuation of one history, a candidate of one step) owns pages
through a row of ``table`` [B, M] int32; a list ``prefix`` of pages lies
before every sequence.  The new tokens of all sequences are packed, sequence
b's at rows starts[b] .. starts[b + 1] - 1 of [N, heads, 128] tensors (starts
[B + 1] int32, from 0 on and not decreasing; None: N / B each).

Every size on the host is a bound only: how many tokens a sequence holds and
where its rows start are read on the device, so a captured call is replayed
with other values.  The attention's work is cut up by those bounds, though: a
table much wider than the sequences are long costs time (64 sequences of up to
600 rows behind 16384: 51 us with 10 pages a row, 123 with 64, 460 with 256).
Nothing here computes on the CPU.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .legacy_components import HEAD_DIM

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_INT, _F64 = torch.int32, torch.float64
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_FAR = 1 << 53                  # positions that float64 counts one by one
_MOST_ROWS = (1 << 30) - 1      # of a sequence, and of a window
_PARTS = {None: 0, True: 1 << 3, False: 2 << 3}        # single_av as the call's flags


# The checks below stand in the path of a call of a few microseconds, so each
# property of a tensor is asked for once and devices are compared by index.

def _overlap(rows, heads, tok, head, size=HEAD_DIM):
    """Whether rows of `size` elements at r * tok + h * head may share elements:
    neither do the heads of a token lie between two tokens, nor the tokens of
    a head between two heads."""
    return (tok < (heads - 1) * head + size and rows > 1 or head < size and heads > 1) and \
        (head < (rows - 1) * tok + size and heads > 1 or tok < size and rows > 1)


def _cache(cache_k, cache_v, dtype, dev):
    """(rows, K/V heads, token stride, head stride) of the resident cache."""
    shape, stride = cache_k.shape, cache_k.stride()
    if cache_k.dtype is not dtype or cache_v.dtype is not dtype:
        raise TypeError("the cache must have the new rows' dtype (bfloat16 or float16)")
    if len(shape) != 4 or cache_v.shape != shape or cache_v.stride() != stride:
        raise ValueError("cache_k and cache_v must be [1, 64P, G, 128] of equal shape and strides")
    one, rows, heads, dim = shape
    _, tok, head, unit = stride
    if one != 1 or dim != HEAD_DIM or rows == 0 or rows & 63 or heads == 0:
        raise ValueError("cache_k and cache_v must be [1, 64P, G, 128]")
    if unit != 1 or (tok | head) & 7 or (cache_k.data_ptr() | cache_v.data_ptr()) & 15 or tok < HEAD_DIM or \
            _overlap(rows, heads, tok, head):
        raise ValueError("the cache's rows must not overlap and must start at multiples of 16 bytes")
    if cache_k.get_device() != dev or cache_v.get_device() != dev:
        raise ValueError("the cache must be on the new rows' device")
    return rows, heads, tok, head


def _rows(x, name, dtype, dev):
    """(N, heads, token stride, head stride, pointer) of packed rows [N, heads, 128]."""
    shape, stride, ptr = x.shape, x.stride(), x.data_ptr()
    if len(shape) != 3 or shape[2] != HEAD_DIM or stride[2] != 1:
        raise ValueError(f"{name} must be [N, heads, 128] with adjacent elements in a row")
    tokens, heads, _ = shape
    tok, head, _ = stride
    if x.dtype is not dtype or x.get_device() != dev:
        raise TypeError(f"{name} must share the other rows' dtype and device")
    if (tok | head) & 7 or ptr & 15:
        raise ValueError(f"{name}'s rows must start at multiples of 16 bytes")
    return tokens, heads, tok, head, ptr


def _written(x, name, dtype, dev):
    """_rows of a tensor that is written: its rows must not overlap."""
    got = _rows(x, name, dtype, dev)
    if _overlap(*got[:4]):
        raise ValueError(f"{name}'s rows must not overlap")
    return got


def _in_place(ptr, tok, head, n, h, start):
    """Whether n x h rows at `ptr` are those of a contiguous tensor at `start`."""
    return ptr == start and (n < 2 or tok == h * HEAD_DIM) and (h < 2 or head == HEAD_DIM)


def _ints(x, name, shape, dev):
    if x.dtype is not _INT or x.shape != shape or not x.is_contiguous() or x.get_device() != dev:
        raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the rows' device")
    return x.data_ptr()


def _sequences(table, starts, tokens, dev):
    """(batch, pages a sequence may own, table pointer, starts pointer)."""
    if table.dim() != 2:
        raise ValueError("table must be [B, M]")
    batch, width = shape = table.shape
    if batch == 0 or width == 0:
        raise ValueError("table must be [B, M]")
    ptr = _ints(table, "table", shape, dev)
    if starts is None:
        if tokens % batch:
            raise ValueError("without starts, the sequences have N / B new tokens each: N must be a multiple of B")
        return batch, width, ptr, None
    return batch, width, ptr, _ints(starts, "starts", (batch + 1,), dev)


def _launch(name, device, dev, *args):
    """The library's entry `name` with `device` current, on its current stream."""
    if dev < 0:
        raise RuntimeError("the tensors must be on a GPU")
    fn = getattr(_lib.lib(), name)
    if dev == torch.cuda.current_device():
        _lib.check(fn(*args, _lib.stream_handle(device)), name)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _lib.stream_handle(device)), name)


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
    are formed in float64: within 2^-24 of a turn up to 2^27 turns, and as
    float64 holds them beyond; `first` lies within 2^53.

    q_out: where the rotated queries go (q itself is allowed; otherwise it must
    not overlap what is read); else a buffer owned by `workspace` that the next
    call, of whatever size, overwrites (so q may be the last call's result as
    it stands, but no other part of that buffer), or, without one, a new tensor."""
    device, dtype, dev = k.device, k.dtype, k.get_device()
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError("k must be bfloat16 or float16")
    if not -_FAR <= first <= _FAR:
        raise ValueError("first must lie within 2^53")
    rows, g, kv_tok, kv_head = _cache(cache_k, cache_v, dtype, dev)
    return _append("ssa_paged_append", (cache_k.data_ptr(), cache_v.data_ptr(), kv_tok, kv_head), rows >> 6, g, k, v,
                   table, held, q, q_out, starts, freqs, axes, positions, first, interleaved, workspace, code)


def _append(entry, cache, pages, gc, k, v, table, held, q, q_out, starts, freqs, axes, positions, first, interleaved,
            workspace, code):
    """append to the cache that the entry takes as `cache`."""
    device, dtype, dev = k.device, k.dtype, k.get_device()
    n, g, k_tok, k_head, k_ptr = _rows(k, "k", dtype, dev)
    nv, gv, v_tok, v_head, v_ptr = _rows(v, "v", dtype, dev)
    if nv != n or gv != g or gc != g:
        raise ValueError("k and v must be [N, G, 128] for the cache's G heads")
    batch, width, table_ptr, starts_ptr = _sequences(table, starts, n, dev)
    held_ptr = _ints(held, "held", (batch,), dev)
    pairs, a0, a1, na, freqs_ptr, pos_ptr = 0, 0, 0, 1, None, None
    if freqs is not None:
        if freqs.dtype is not _F64 or freqs.dim() != 1 or freqs.get_device() != dev or not freqs.is_contiguous():
            raise ValueError("freqs must be a contiguous float64 [R] tensor on the rows' device")
        pairs, freqs_ptr = freqs.shape[0], freqs.data_ptr()
        if pairs > HEAD_DIM // 2 or (not interleaved and pairs % 8):
            raise ValueError("at most 64 pairs, a multiple of 8 in halves")
        if axes is None:
            a0 = pairs
        else:
            na = len(axes)
            if not 1 <= na <= 3 or sum(axes) != pairs or min(axes) < 0:
                raise ValueError("axes must be 1 to 3 counts that sum to the pairs")
            a0, a1 = axes[0], axes[1] if na > 1 else 0
        if positions is not None:
            pos_ptr = _ints(positions, "positions", (n,) if na == 1 and positions.dim() == 1 else (n, na), dev)
        elif na > 1:
            raise ValueError("several axes need positions")
    elif positions is not None or axes is not None:
        raise ValueError("positions and axes need freqs")
    h, q_ptr, out_ptr, q_tok, q_head, o_tok, o_head = 0, None, None, 0, 0, 0, 0
    if q is not None:
        nq, h, q_tok, q_head, q_ptr = _rows(q, "q", dtype, dev)
        if nq != n or h == 0:
            raise ValueError("q must be [N, H, 128]")
        if q_out is None:
            o_tok, o_head = h * HEAD_DIM, HEAD_DIM
            if workspace is None:
                q_out = torch.empty((n, h, HEAD_DIM), dtype=dtype, device=device)
                out_ptr = q_out.data_ptr()
            else:
                q_out, out_ptr, end = workspace.rows('paged_q', (n, h, HEAD_DIM), device, dtype)
                if out_ptr <= k_ptr < end or out_ptr <= v_ptr < end or \
                        out_ptr <= q_ptr < end and not _in_place(q_ptr, q_tok, q_head, n, h, out_ptr):
                    raise ValueError("q, k or v lies in the workspace's buffer for the rotated queries: give q_out")
        else:
            no, ho, o_tok, o_head, out_ptr = _written(q_out, "q_out", dtype, dev)
            if no != n or ho != h:
                raise ValueError("q_out must have q's shape")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if n:
        _launch(entry, device, dev, q_ptr, q_tok, q_head, out_ptr, o_tok, o_head, k_ptr, k_tok, k_head, v_ptr, v_tok,
                v_head, *cache, table_ptr, held_ptr, starts_ptr, pos_ptr, freqs_ptr, first, n, batch, h, g, pages,
                width, pairs, a0, a1, na, code | 2 if interleaved else code)
    return q_out


# Workspace bytes by sizes and device, rounded up to a power of two: calls of many
# sizes share a few buffers.
_BYTES = {}


def attention(q, cache_k, cache_v, prefix, prefix_tokens, table, lengths, workspace, *, starts=None, causal=True,
              scale=None, want_lse=False, out=None, single_av=None, cap=None, slopes=None, window=None):
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
    as they were.  Pages outside the cache (-1) and, where a length passes it,
    behind the table's end count as absent; rows that no query sees may hold
    anything, while a value row that some query of the call sees must be
    finite for the others to come out finite (an infinite one may come out NaN).

    scale defaults to 128 ** -0.5.  Returns out [N, H, 128], or (out, lse)
    with want_lse, lse [N, H] float32 the log of the sum of exponentials:
    buffers owned by `workspace` and overwritten by the next call, of whatever
    size, or `out` as given (q itself is allowed; otherwise it must not overlap
    what is read).

    Arithmetic: scores, maxima, sums and the joins of pieces are float32.  A
    probability meets V in 16 bits (fp16: scaled up by 2^7): in two parts (hi
    + lo), which leave the output its own rounding, or in one, with which its
    error is 1.4 times as large.  ``single_av=False``: two parts throughout;
    the default None: two where the sequences bring up to 32 rows a K/V head
    (their mean: new tokens times H / G), else one in tiles of more than 32
    rows, which the matrix pipe bounds (two parts take 1.4 times as long
    there); ``single_av=True``: one in all tiles of more than 32 rows.  Sums
    reach 2^8 times the values' size times the rows: bf16 values from 2^96 on,
    and fp16 values within 2^-11 of the type's largest, may come out infinite.

    Shaped scores, each for itself or together, of s = scale q.k:
    cap (up to 65536, not so small that 2 log2(e) scale / cap overflows float32): s
    becomes cap tanh(s / cap), within 2^-22 of the cap;
    slopes [H] float32, finite: s falls by the head's slope times the distance in rows
    between query and key, query i's own row being lengths[b] - n + i and the
    prefix's rows lying before row 0 (keys behind the query count alike), within
    2^-22 of the fall, which must be finite in float32;
    window (1 or more): of its own sequence a query sees only the `window` rows up
    to its own (without `causal` also those behind it), and all of the prefix.
    Pages that no query sees any more may be absent, and are not walked."""
    code = _TYPES.get(q.dtype)
    if code is None:
        raise TypeError("q must be bfloat16 or float16")
    dev = q.get_device()
    rows, g, kv_tok, kv_head = _cache(cache_k, cache_v, q.dtype, dev)
    return _attend("ssa_paged_attention", False, (cache_k.data_ptr(), cache_v.data_ptr(), kv_tok, kv_head), rows >> 6,
                   g, q, prefix, prefix_tokens, table, lengths, workspace, starts, causal, scale, want_lse, out,
                   single_av, cap, slopes, window, code)


def _shape(cap, slopes, window, heads, dev):
    """The entries' cap, slopes and window."""
    if cap is None:
        cap = 0.0
    elif not 2.0 ** -126 <= cap <= 65536.0:
        raise ValueError("cap must be positive, 65536 at most")
    slopes_ptr = None
    if slopes is not None:
        if slopes.dtype is not torch.float32 or slopes.shape != (heads,) or not slopes.is_contiguous() or \
                slopes.get_device() != dev:
            raise ValueError("slopes must be a contiguous float32 [H] tensor on the rows' device")
        slopes_ptr = slopes.data_ptr()
    if window is None:
        window = 0
    elif not 1 <= window < math.inf or window != int(window):
        raise ValueError("window must be a whole number from 1 on")
    return cap, slopes_ptr, min(int(window), _MOST_ROWS)


def _attend(entry, eight, cache, pages, g, q, prefix, prefix_tokens, table, lengths, workspace, starts, causal, scale,
            want_lse, out, single_av, cap, slopes, window, code):
    """attention over the cache that the entry takes as `cache`."""
    device, dtype, dev = q.device, q.dtype, q.get_device()
    n, h, q_tok, q_head, q_ptr = _rows(q, "q", dtype, dev)
    if h == 0 or h % g:
        raise ValueError("the query heads must be a multiple of the cache's heads")
    batch, width, table_ptr, starts_ptr = _sequences(table, starts, n, dev)
    len_ptr = _ints(lengths, "lengths", (batch,), dev)
    prefix_ptr = None
    if prefix_tokens > 0:
        if prefix is None or prefix.dim() != 1 or prefix.shape[0] << 6 < prefix_tokens:
            raise ValueError("prefix must list the pages of prefix_tokens rows")
        prefix_ptr = _ints(prefix, "prefix", prefix.shape, dev)
    elif prefix_tokens < 0:
        raise ValueError("prefix_tokens must not be negative")
    parts = _PARTS.get(single_av)
    if parts is None:
        raise ValueError("single_av must be None, True or False")
    if scale is None:
        scale = _SCALE
    elif not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive")
    if out is None:
        out, out_ptr, end = workspace.rows('paged_out', (n, h, HEAD_DIM), device, dtype)
        o_tok, o_head = h * HEAD_DIM, HEAD_DIM
        if out_ptr <= q_ptr < end and not _in_place(q_ptr, q_tok, q_head, n, h, out_ptr):
            raise ValueError("q lies in the workspace's buffer for the output: give out")
    else:
        no, ho, o_tok, o_head, out_ptr = _written(out, "out", dtype, dev)
        if no != n or ho != h:
            raise ValueError("out must have q's shape")
    lse = lse_ptr = None
    if want_lse:
        lse, lse_ptr, _ = workspace.rows('paged_lse', (n, h), device, torch.float32)
    shape = ()
    if cap is not None or slopes is not None or window is not None:
        shape = _shape(cap, slopes, window, h, dev)
        entry += "_shaped"
    if n:
        key = (n, batch, h, g, prefix_tokens, width, starts is None, causal, dev)
        if eight or shape:
            key += (eight, bool(shape), shape[2] if shape else 0)
        need = _BYTES.get(key)
        if need is None:
            need = _workspace_bytes(key, device)
        part = workspace.tensor('paged_part', (need,), device, torch.uint8).data_ptr() if need else None
        _launch(entry, device, dev, q_ptr, q_tok, q_head, *cache, prefix_ptr, prefix_tokens, table_ptr, len_ptr,
                starts_ptr, out_ptr, o_tok, o_head, lse_ptr, n, batch, h, g, pages, width, scale, *shape,
                (code | 2 if causal else code) | parts, part, need)
    return (out, lse) if want_lse else out


def _workspace_bytes(key, device):
    """The workspace of a call of these sizes, asked of the library once per sizes
    and device."""
    tokens, batch, heads, kv_heads, prefix_tokens, width, equal, causal, dev, *form = key
    if dev < 0:
        raise RuntimeError("the tensors must be on a GPU")
    eight, shaped, window = form or (False, False, 0)
    with torch.cuda.device(device):
        need = _lib.lib().ssa_paged8_workspace_bytes(tokens, batch, heads, kv_heads, prefix_tokens, width,
                                                     int(not equal), int(bool(causal)), int(eight), int(shaped), window)
    if need < 0:
        raise ValueError("paged.attention: sizes out of range")
    if need:
        need = 1 << (need - 1).bit_length()
    if len(_BYTES) >= 4096:
        _BYTES.clear()
    _BYTES[key] = need
    return need
