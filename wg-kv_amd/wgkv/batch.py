"""Serving a packed batch of requests over paged per-head caches.

A step's tokens of B requests lie behind each other in packed tensors, request
b's at rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` (int32, ascending).
Caches are the pools ``(num_blocks, block_size, head_dim)`` bf16, page tables
``(batch, num_kv_heads, max_blocks)`` and lengths ``(batch, num_kv_heads)`` of
``paged_decode_attn``.

    lengths, slots, pages = build_block_tables(...)   pages, lengths and rows of a step's tokens
    paged_append(k, v, k_cache, v_cache, slots)       the tokens' keys and values to those rows
    sink_window_attn(...)                             prompts: a sliding window and first tokens
    paged_decode_attn_window(...)                     the same for one token over the cache
    paged_decode_attn_shared(...)                     one token over a prefix that sequences share

The operators run on torch's current stream of the tensors' device, allocate
only their outputs and scratch (both through torch, so a call can be captured
in a HIP graph) and never synchronise with the host.  A tensor they write must
not overlap itself or, but for build_block_tables' lengths and page state in
place, one they read.
"""
import functools
import struct

import torch

from . import _lib
from .kv4 import _attn_workspace, _check_heads, _current_device, _host_tensor, _rows, _stream, _two_devices
from .ops import _u8

_I32, _U8, _BF16 = torch.int32, torch.uint8, torch.bfloat16
# arguments of the C calls as blocks of 8-byte words (wgkv_*_block)
_pack_tables = struct.Struct("25q").pack
_pack_append = struct.Struct("14q").pack
_pack_prompt = struct.Struct("22qd4q").pack
_pack_window = struct.Struct("22qd3q").pack
_pack_shared = struct.Struct("28qd3q").pack
_MOST = 2 ** 31 - 1


def _check_pool(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 3 or v_cache.shape != shape:
        raise AssertionError("k_cache/v_cache must be (num_blocks, block_size, head_dim)")
    if k_cache.dtype is not _BF16 or v_cache.dtype is not _BF16:
        raise TypeError("k_cache/v_cache must be bf16")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous")
    return shape


def _check_starts(cu, what):
    """A vector of ascending row numbers, with its number of ranges."""
    if cu.dim() != 1 or cu.shape[0] < 2:
        raise AssertionError(f"{what} must be one entry more than its ranges, of which there is one at least")
    if cu.dtype is not _I32:
        raise TypeError(f"{what} must be int32")
    return cu if cu.stride(0) == 1 else cu.contiguous(), cu.shape[0] - 1


def _same_device(dev, *tensors):
    if dev < 0:
        _host_tensor()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _two_devices()


def _rows3(t, copy=True):
    """t (rows, heads, d), its address and strides if its rows can be read and
    written 16 bytes at a time, else (``copy``) a contiguous copy's, or None."""
    st = t.stride()
    p = t.data_ptr()
    a = 0 if t.shape[0] == 1 else st[0]  # the stride of a dimension of one entry means nothing
    b = 0 if t.shape[1] == 1 else st[1]
    if st[2] == 1 and not (a | b) % 8 and not p % 16:
        return t, p, (a, b)
    if not copy:
        return None
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.stride()


def build_block_tables(lengths, cu_seqlens, num_tokens, block_table, page_state, num_blocks, block_size, g_mask=None,
                       free_ids=None, out=None, state_out=None, slots=None, status=None):
    """Pages, lengths and cache rows of a step's ``num_tokens`` packed tokens.

    Head (b, h) holds ``lengths[b, h]`` tokens and takes those of request b
    that ``g_mask`` (num_kv_heads, num_tokens) keeps -- all without it -- to its
    next positions.  The pages they need come, heads in (b, h) order, from the
    last entries of ``free_ids`` (int32, optional) in list order, then from the
    next unused page on; ``page_state`` (int32 (2,)) is that page and the
    number of entries the list holds.  Their ids are written to
    ``block_table`` (int32 (batch, num_kv_heads, max_blocks), in place); its
    other entries stay.

    Returns (new lengths, slots, new page state): slots int32 (num_tokens,
    num_kv_heads) are rows of the pools, ``page * block_size + position %
    block_size``, and -1 for tokens that are not kept or belong to no request.
    ``out`` may be ``lengths`` and ``state_out`` may be ``page_state`` itself.

    If the pages of the pool's ``num_blocks`` do not suffice, or a head would
    outgrow its table, the step is refused as a whole: the table, the lengths
    and the state stay, slots are -1 and ``status`` (int32, optional) is set to
    WGKV_ERR_CAPACITY.  A held page id outside the pool sets it too, and its
    tokens' slots are -1.
    """
    if block_table.dim() != 3:
        raise AssertionError("block_table must be (batch, num_kv_heads, max_blocks)")
    B, H, width = block_table.shape
    cu, ranges = _check_starts(cu_seqlens, "cu_seqlens")
    if ranges != B:
        raise AssertionError("cu_seqlens must have batch + 1 entries")
    table, bs, _, lens, ls = _check_heads(block_table, lengths, B, H)
    if table is not block_table:
        raise ValueError("block_table is written in place: its last dimension must be contiguous")
    if num_tokens < 0:
        raise AssertionError("num_tokens must not be negative")
    if g_mask is not None and g_mask.shape != (H, num_tokens):
        raise AssertionError("g_mask must be (num_kv_heads, num_tokens)")
    for t, name in ((page_state, "page_state"), (state_out, "state_out")):
        if t is not None and (t.shape != (2,) or t.dtype is not _I32 or not t.is_contiguous()):
            raise AssertionError(f"{name} must be int32 (2,)")
    if free_ids is not None and (free_ids.dim() != 1 or free_ids.dtype is not _I32 or not free_ids.is_contiguous()):
        raise AssertionError("free_ids must be a contiguous int32 vector")
    if out is not None and (out.shape != (B, H) or out.dtype is not _I32 or (H > 1 and out.stride(1) != 1)):
        raise AssertionError("out must be int32 (batch, num_kv_heads), heads contiguous")
    if slots is not None and (slots.shape != (num_tokens, H) or slots.dtype is not _I32 or not slots.is_contiguous()):
        raise AssertionError("slots must be contiguous int32 (num_tokens, num_kv_heads)")
    if status is not None and (status.dtype is not _I32 or status.numel() < 1):
        raise TypeError("status must be an int32 tensor")
    dev = block_table.get_device()
    _same_device(dev, lens, cu, g_mask, page_state, state_out, free_ids, out, slots, status)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return build_block_tables(lengths, cu_seqlens, num_tokens, block_table, page_state, num_blocks, block_size,
                                      g_mask, free_ids, out, state_out, slots, status)
    mp = ms = 0
    if g_mask is not None:
        m = _u8(g_mask)
        if num_tokens > 1 and m.stride(1) != 1:
            m = m.contiguous()
        mp, ms = m.data_ptr(), m.stride(0)
    if out is None:
        out = torch.empty_like(lens, memory_format=torch.contiguous_format)
    if slots is None:
        slots = lens.new_empty((num_tokens, H))
    if state_out is None:
        state_out = torch.empty_like(page_state)
    L = _lib.lib()
    free, held = (free_ids.data_ptr(), free_ids.shape[0]) if free_ids is not None and free_ids.shape[0] else (0, 0)
    args = (
        lens.data_ptr(), ls, cu.data_ptr(), num_tokens, mp, ms, table.data_ptr(), bs[0], bs[1], width,
        page_state.data_ptr(), state_out.data_ptr(), free, held, num_blocks, block_size, out.data_ptr(), out.stride(0),
        slots.data_ptr(), B, H, 0 if status is None else status.data_ptr())
    st = _lib.ERR_WORKSPACE
    if num_tokens <= 256 or not mp:  # (most of these need no scratch)
        st = L.wgkv_build_block_tables_block(_pack_tables(*args, 0, 0, _stream(dev)))
    if st == _lib.ERR_WORKSPACE:
        ws = torch.empty(L.wgkv_block_tables_workspace_bytes(B, H, num_tokens), dtype=_U8, device=dev)
        st = L.wgkv_build_block_tables_block(_pack_tables(*args, ws.data_ptr(), ws.numel(), _stream(dev)))
    if st:
        _lib.check(st, "wgkv_build_block_tables")
    return out, slots, state_out


def paged_append(k, v, k_cache, v_cache, slots):
    """Copies the rows of k, v (tokens, num_kv_heads, head_dim) bf16, in any
    layout, to rows ``slots[n, h]`` (int32) of the pools; slots outside them
    (-1) are left out.  The slots in them are to differ, as those of
    build_block_tables do where no page stands in the tables twice: tokens that
    share one leave rows in which each 8 values are one token's, but not all the
    same token's, and not the same in every call."""
    shape = k.shape
    pool = _check_pool(k_cache, v_cache)
    if len(shape) != 3 or v.shape != shape or shape[2] != pool[2]:
        raise AssertionError("k/v must be (tokens, num_kv_heads, head_dim)")
    if k.dtype is not _BF16 or v.dtype is not _BF16:
        raise TypeError("k/v must be bf16")
    if slots.shape != shape[:2]:
        raise AssertionError("slots must be (tokens, num_kv_heads)")
    if slots.dtype is not _I32:
        raise TypeError("slots must be int32")
    dev = k_cache.get_device()
    _same_device(dev, v_cache, k, v, slots)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_append(k, v, k_cache, v_cache, slots)
    if not shape[0]:
        return
    k, kp, ks = _rows3(k)
    v, vp, vs = _rows3(v)
    if not slots.is_contiguous():
        slots = slots.contiguous()
    st = _lib.lib().wgkv_paged_append_block(_pack_append(
        kp, ks[0], ks[1], vp, vs[0], vs[1], k_cache.data_ptr(), v_cache.data_ptr(), pool[0] * pool[1], slots.data_ptr(),
        shape[0], shape[1], shape[2], _stream(dev)))
    if st:
        _lib.check(st, "wgkv_paged_append")


def sink_window_attn(q, k, v, cu_seqlens, window, num_sinks, softmax_scale=None, cu_seqlens_k=None, out=None):
    """Causal attention of a packed batch of prompts in which a row sees a
    sliding window and the first tokens of its sequence.

    q (rows, Hq, D), k and v (keys, Hkv, D) bf16 in any layout, D 64 or 128,
    Hq / Hkv from 1 to 8; sequence b holds the rows ``cu_seqlens[b] ..`` and the
    keys ``cu_seqlens_k[b] ..`` (without it: the same).  With nq rows and nk
    keys its row i is at position p = i + nk - nq (the rows are the last of its
    keys) and sees key j if j <= p and (j > p - window or j < num_sinks);
    ``window`` counts the row's own key.  Rows that see nothing give zeros.  Keys
    and values are dense, those of earlier chunks too; pages are not read.

    Returns (rows, Hq, D) bf16; rows of no sequence are zeros, or left as they
    are in a given ``out``.  Probabilities are rounded to bf16 for the products;
    sums are fp32, before their division by the probabilities' sum.  What a row
    does not see has no part in its result, whatever it holds; what it sees has,
    with a weight of 0 too (0 times infinity is NaN).  Up to 2048 sequences.

    Rows next to those that see a value that is not finite are worked out on their
    own: 0.12 ms per 1000 keys, up to 32 of them one after the other.
    """
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3 or v.shape != kshape or kshape[2] != shape[2]:
        raise AssertionError("q must be (rows, num_query_heads, head_dim), k/v (keys, num_kv_heads, head_dim)")
    N, Hq, D = shape
    Nk, H, _ = kshape
    if H < 1 or Hq < 1 or Hq % H:
        raise AssertionError("num_query_heads must be a multiple of num_kv_heads")
    if q.dtype is not _BF16 or k.dtype is not _BF16 or v.dtype is not _BF16:
        raise TypeError("q, k and v must be bf16")
    cu, B = _check_starts(cu_seqlens, "cu_seqlens")
    cuk = cu
    if cu_seqlens_k is not None and cu_seqlens_k is not cu_seqlens:
        cuk, ranges = _check_starts(cu_seqlens_k, "cu_seqlens_k")
        if ranges != B:
            raise AssertionError("cu_seqlens and cu_seqlens_k must have one length")
    if window < 1 or num_sinks < 0:
        raise ValueError("window must be positive and num_sinks not negative")
    dev = q.get_device()
    _same_device(dev, k, v, cu, cuk, out)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return sink_window_attn(q, k, v, cu_seqlens, window, num_sinks, softmax_scale, cu_seqlens_k, out)
    if softmax_scale is None:
        softmax_scale = D ** -0.5
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not _BF16:
        raise AssertionError("out must be (rows, num_query_heads, head_dim) bf16")
    if not N:
        return out
    rows = _rows3(out, False)
    if rows is None:  # they cannot be written 16 bytes at a time
        tmp = out.clone(memory_format=torch.contiguous_format)  # (keeps the rows of no sequence)
        return out.copy_(sink_window_attn(q, k, v, cu, window, num_sinks, softmax_scale, cuk, tmp))
    _, op, os = rows
    q, qp, qs = _rows3(q)
    k, kp, ks = _rows3(k)
    v, vp, vs = _rows3(v)
    window, num_sinks = min(window, _MOST), min(num_sinks, _MOST)
    L = _lib.lib()
    args = (
        qp, qs[0], qs[1], kp, ks[0], ks[1], vp, vs[0], vs[1], op, os[0], os[1], cu.data_ptr(), cuk.data_ptr(), B, N, Nk,
        Hq, H, D, window, num_sinks, softmax_scale, not given)
    st = L.wgkv_sink_window_attn_block(_pack_prompt(*args, 0, 0, _stream(dev)))
    if st == _lib.ERR_WORKSPACE:  # few rows behind many keys; others are spared the question (1 us)
        ws = torch.empty(L.wgkv_sink_window_workspace_bytes(B, N, Nk, Hq, H, D, window, num_sinks), dtype=_U8, device=dev)
        st = L.wgkv_sink_window_attn_block(_pack_prompt(*args, ws.data_ptr(), ws.numel(), _stream(dev)))
    if st:
        _lib.check(st, "wgkv_sink_window_attn")
    return out


def _check_token(q, cache_seqlens, block_table, pool):
    """One query row per sequence over a paged cache."""
    shape = q.shape
    if len(shape) != 4 or shape[1] != 1 or shape[3] != pool[2]:
        raise AssertionError("q must be (batch, 1, num_query_heads, head_dim)")
    if q.dtype is not _BF16:
        raise TypeError("q must be bf16")
    H = cache_seqlens.shape[1] if cache_seqlens.dim() == 2 else -1
    heads = _check_heads(block_table, cache_seqlens, shape[0], H)
    if H < 1 or shape[2] % H:
        raise AssertionError("num_query_heads must be a multiple of num_kv_heads")
    return shape, H, heads


def _token_out(q, out):
    """The output of a call with one row per sequence, its address and strides."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype is not _BF16:
        raise AssertionError("out must be (batch, 1, num_query_heads, head_dim) bf16")
    st = out.stride()
    return (out, out.data_ptr(), st) if st[3] == 1 else None


@functools.lru_cache(maxsize=1024)
def _window_bytes(B, Hq, H, D):
    return _lib.lib().wgkv_paged_decode_window_workspace_bytes(B, Hq, H, D)


def paged_decode_attn_window(q, k_cache, v_cache, cache_seqlens, block_table, window, num_sinks, softmax_scale, out=None):
    """``paged_decode_attn`` over a sliding window and the first tokens: q (B,
    1, Hq, D) bf16 attends, of the T = cache_seqlens[b, h] tokens of its KV
    head, to those t with t >= T - window or t < num_sinks (the newest token
    counts to the window; where a gate left tokens out, these are the head's kept
    tokens, not the positions that sink_window_attn counts); returns (B, 1, Hq, D) bf16, zeros for a head without
    tokens.  Pages that hold none of them are not read, and their table
    entries may be anything: they can be given back.  Unlike there, a NaN or +inf
    among the scores that a head sees makes its result NaN.  Hq / Hkv up to 8, B * Hkv
    up to 2048.  Lengths and page ids out of range are clamped to the table
    and the pool."""
    pool = _check_pool(k_cache, v_cache)
    shape, H, (table, bs, width, lens, ls) = _check_token(q, cache_seqlens, block_table, pool)
    if window < 1 or num_sinks < 0:
        raise ValueError("window must be positive and num_sinks not negative")
    B, _, Hq, D = shape
    dev = q.get_device()
    _same_device(dev, k_cache, v_cache, lens, table, out)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_decode_attn_window(q, k_cache, v_cache, cache_seqlens, block_table, window, num_sinks,
                                            softmax_scale, out)
    rows = _token_out(q, out)
    if rows is None:
        return out.copy_(paged_decode_attn_window(q, k_cache, v_cache, lens, table, window, num_sinks, softmax_scale))
    out, op, os = rows
    q, qp, qs = _rows(q, 8)
    stream = _stream(dev)
    ws = _attn_workspace(dev, stream, _window_bytes(B, Hq, H, D))
    st = _lib.lib().wgkv_paged_decode_attn_window_block(_pack_window(
        qp, qs[0], qs[2], k_cache.data_ptr(), v_cache.data_ptr(), pool[0], pool[1], lens.data_ptr(), ls,
        table.data_ptr(), bs[0], bs[1], width, op, os[0], os[2], B, Hq, H, D, min(window, _MOST), min(num_sinks, _MOST),
        softmax_scale, ws.data_ptr(), ws.numel(), stream))
    if st:
        _lib.check(st, "wgkv_paged_decode_attn_window")
    return out


@functools.lru_cache(maxsize=1024)
def _shared_bytes(B, N, Hq, H, D):
    return _lib.lib().wgkv_shared_decode_workspace_bytes(B, N, Hq, H, D)


def paged_decode_attn_shared(q, k_cache, v_cache, cache_seqlens, block_table, prefix_lens, prefix_table, group_starts,
                             softmax_scale, out=None):
    """``paged_decode_attn`` of a batch whose sequences share prefixes, each
    prefix read for many rows of its group at once: for 16 (sequence, query head
    of a KV head) where groups have up to 16 on average, otherwise for 256.

    Sequences ``group_starts[n] .. group_starts[n + 1] - 1`` (int32, ascending;
    N + 1 entries) share prefix n: each of their heads attends to the first
    ``prefix_lens[n, h]`` (int32 (N, Hkv)) tokens of the pages ``prefix_table[n,
    h]`` (int32 (N, Hkv, prefix_blocks)) and to the first cache_seqlens[b, h]
    tokens of its own pages, under one softmax.  Sequences outside
    [group_starts[0], group_starts[N]) have no prefix.  q (B, 1, Hq, D) bf16;
    returns (B, 1, Hq, D) bf16, zeros for a head without tokens.  Hq / Hkv up to
    8, B * Hkv and N * Hkv up to 2048.  Probabilities are rounded to bf16 for
    their product with the values; sums are fp32.  Lengths and page ids out of
    range are clamped to the tables and the pool."""
    pool = _check_pool(k_cache, v_cache)
    shape, H, (table, bs, width, lens, ls) = _check_token(q, cache_seqlens, block_table, pool)
    starts, N = _check_starts(group_starts, "group_starts")
    ptable, ps, pwidth, plens, pls = _check_heads(prefix_table, prefix_lens, N, H)
    B, _, Hq, D = shape
    dev = q.get_device()
    _same_device(dev, k_cache, v_cache, lens, table, plens, ptable, starts, out)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_decode_attn_shared(q, k_cache, v_cache, cache_seqlens, block_table, prefix_lens, prefix_table,
                                            group_starts, softmax_scale, out)
    rows = _token_out(q, out)
    if rows is None:
        return out.copy_(paged_decode_attn_shared(q, k_cache, v_cache, lens, table, plens, ptable, starts,
                                                  softmax_scale))
    out, op, os = rows
    q, qp, qs = _rows(q, 8)
    nbytes = _shared_bytes(B, N, Hq, H, D)
    ws = torch.empty(nbytes, dtype=_U8, device=dev)
    st = _lib.lib().wgkv_shared_decode_attn_block(_pack_shared(
        qp, qs[0], qs[2], k_cache.data_ptr(), v_cache.data_ptr(), pool[0], pool[1], lens.data_ptr(), ls,
        table.data_ptr(), bs[0], bs[1], width, plens.data_ptr(), pls, ptable.data_ptr(), ps[0], ps[1], pwidth,
        starts.data_ptr(), N, op, os[0], os[2], B, Hq, H, D, softmax_scale, ws.data_ptr(), nbytes, _stream(dev)))
    if st:
        _lib.check(st, "wgkv_shared_decode_attn")
    return out
